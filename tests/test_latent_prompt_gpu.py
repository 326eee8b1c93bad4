"""Latent attention, expanded form, against a 64-bit reference (bounds: see test_latent_gpu)."""

import math

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.verify_ref import _weigh, attention_bound
from torch_spyre_b200 import _lib

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Case:
    def __init__(self, new, lens, heads, dtype=BF16, causal=True, seed=0, qscale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n, m = sum(new), sum(lens)

        def randn(*shape):
            return torch.randn(shape, generator=g, device="cuda")

        self.new, self.lens, self.heads, self.causal = new, lens, heads, causal
        self.q = (randn(n, heads, 192) * qscale).to(dtype)
        kv = randn(m, heads, 256).to(dtype)
        self.k_nope, self.v = kv[..., :128], kv[..., 128:]
        self.k_rope = randn(m, 576).to(dtype)[:, 512:]
        ptr = lambda x: torch.tensor([0] + torch.tensor(x, dtype=torch.int64).cumsum(0).tolist(), dtype=torch.int32,  # noqa: E731
                                     device="cuda")
        self.q_indptr, self.kv_indptr = ptr(new), ptr(lens)

    def args(self):
        return self.q, self.k_nope, self.k_rope, self.v, self.q_indptr, self.kv_indptr

    def reference(self, scale=None):
        scale = 192**-0.5 if scale is None else scale
        outs, lses, spreads, a, c = [], [], [], 0, 0
        for n, m in zip(self.new, self.lens):
            q, k = self.q[a:a + n].double(), self.k_nope[c:c + m].double()
            k = torch.cat([k, self.k_rope[c:c + m, None].double().expand(m, self.heads, 64)], -1)
            v = self.v[c:c + m].double()
            s = torch.einsum("thd,phd->htp", q, k) * scale
            see = torch.ones(n, m, dtype=torch.bool, device="cuda")
            if self.causal:
                see = torch.arange(m, device="cuda") <= m - n + torch.arange(n, device="cuda")[:, None]
            s = s.masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, -1) if m else torch.full((self.heads, n), -math.inf, device="cuda", dtype=torch.float64)
            w = torch.where(see & (lse[..., None] > -math.inf), torch.exp(s - lse[..., None]), 0.0)
            outs.append(_weigh(w, v))
            spreads.append(_weigh(w, v.abs()))
            lses.append(lse.transpose(0, 1))
            a, c = a + n, c + m
        return torch.cat(outs), torch.cat(lses), torch.cat(spreads)


def check(case, **kw):
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = tsb.latent_prompt_attention(*case.args(), causal=case.causal, return_lse=True, error_flag=flag, **kw)
    assert int(flag.item()) == 0
    ref, ref_lse, spread = case.reference(kw.get("scale"))
    bound = attention_bound(ref, spread, max(case.lens), out.dtype)
    err = (out.double() - ref).abs()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert bool(((err <= bound) | torch.isnan(ref) | (out.double() == ref)).all()), \
        f"off by {float((err / bound).nan_to_num().max()):.3g} of the bound"
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((out[empty] == 0).all())
    assert bool(((lse.double() - ref_lse).abs() <= 2e-4 * (1 + ref_lse.abs()))[~empty].all())
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,past", [([1], [0]), ([1], [300]), ([5, 128, 129, 127], [0, 0, 0, 0]), ([256, 257, 300], [0, 1, 63]),
                                      ([3, 0, 700, 64, 1], [200, 5, 0, 1000, 0]), ([1025], [777])])
def test_lengths(dtype, causal, new, past):
    check(Case(new, [p + n for p, n in zip(past, new)], 3, dtype, causal, seed=sum(new)))


@pytest.mark.parametrize("heads", [1, 2, 16, 128])
def test_heads(heads):
    check(Case([70, 300], [70, 333], heads, seed=heads))


def test_more_rows_than_tokens():
    # the first rows of a sequence see nothing, nor does one without tokens
    check(Case([10, 300, 5, 200], [4, 40, 0, 199], 2, seed=1))
    check(Case([10, 3], [0, 0], 2, seed=1))
    check(Case([10, 300, 5], [4, 40, 0], 2, causal=False, seed=1))


def test_many_sequences():
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 40, (400,), generator=g).tolist()
    past = torch.randint(0, 90, (400,), generator=g).tolist()
    check(Case(new, [p + n for p, n in zip(past, new)], 2, seed=7))
    check(Case([1] * 1024, [3] * 1024, 1, seed=8))


def test_long_pasts_are_split():
    check(Case([3], [30003], 2, F16, seed=3))
    check(Case([200], [20000], 1, BF16, seed=4))
    check(Case([600], [9000], 2, BF16, causal=False, seed=5))


def test_large_scores_and_rising_maxima():
    check(Case([200, 64], [900, 64], 2, qscale=20.0, seed=14))
    case = Case([300], [1500], 2, F16, seed=15)
    ramp = torch.linspace(0.1, 6.0, 1500, device="cuda")
    case.k_nope = (case.q[0, :, :128].float() * ramp[:, None, None]).half()
    check(case)


@pytest.mark.parametrize("scale", [0.4, -0.05, 0.0])
def test_scales(scale):
    check(Case([100, 30], [120, 30], 2, F16, seed=16), scale=scale)


def test_strides():
    case = Case([100, 130], [100, 200], 4, seed=17)
    first = check(case)
    for name in ("q", "k_nope", "v"):
        x = getattr(case, name)
        across = torch.empty((x.shape[1], x.shape[0], x.shape[2] + 8), dtype=x.dtype, device="cuda")[..., :x.shape[2]]
        across.copy_(x.transpose(0, 1))
        setattr(case, name, across.transpose(0, 1))
    case.k_rope = case.k_rope.contiguous()
    assert torch.equal(check(case), first)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,past", [([300, 40], [0, 100]), ([100], [70])])
def test_non_finite_values_reach_the_rows_that_see_them(value, new, past):
    for at in (60, 200):
        case = Case(new, [p + n for p, n in zip(past, new)], 2, seed=18)
        if at < case.v.shape[0]:
            case.v[at, 1, 9] = value
            check(case)


def test_another_sequences_tokens_do_not_matter():
    case = Case([100, 50], [100, 50], 2, seed=19)
    first = tsb.latent_prompt_attention(*case.args())
    for t in (case.k_nope, case.v):
        t[100:] = float("nan")
    out = tsb.latent_prompt_attention(*case.args())
    assert torch.equal(out[:100], first[:100]) and bool(torch.isnan(out[100:]).any())


def test_bad_offsets_are_flagged():
    case = Case([100, 50], [100, 60], 2, seed=20)
    int32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for q_ptr, kv_ptr in (((0, 100, 149), None), ((0, 100, 151), None), ((1, 100, 150), None), (None, (0, 100, 161)),
                          (None, (-1, 100, 160))):
        flag = int32(0)
        out = tsb.latent_prompt_attention(case.q, case.k_nope, case.k_rope, case.v,
                                          case.q_indptr if q_ptr is None else int32(*q_ptr),
                                          case.kv_indptr if kv_ptr is None else int32(*kv_ptr), error_flag=flag)
        assert int(flag) == _lib.DEVERR_BAD_LEN and bool(torch.isfinite(out).all())
    for q_ptr, kv_ptr in (((0, 200, 150), (0, 100, 160)), ((0, 100, 150), (0, 160, 100))):
        flag = int32(0)
        out, lse = tsb.latent_prompt_attention(case.q, case.k_nope, case.k_rope, case.v, int32(*q_ptr), int32(*kv_ptr),
                                               return_lse=True, error_flag=flag)
        assert int(flag) == _lib.DEVERR_BAD_LEN and not out.any() and bool((lse == -math.inf).all())


def test_chunk_and_past_are_joined():
    """A chunk's own tokens (causal) and its past (not causal), merged, are the whole."""
    case = Case([150], [700], 4, F16, seed=22)
    whole, whole_lse = tsb.latent_prompt_attention(*case.args(), return_lse=True)
    past, own = slice(0, 550), slice(550, 700)
    outs, lses = [], []
    for part, causal in ((past, False), (own, True)):
        m = torch.tensor([0, part.stop - part.start], dtype=torch.int32, device="cuda")
        o, x = tsb.latent_prompt_attention(case.q, case.k_nope[part], case.k_rope[part], case.v[part], case.q_indptr, m,
                                           causal=causal, return_lse=True)
        outs.append(o)
        lses.append(x)
    merged, lse = tsb.merge_attention_states(outs, lses)
    # two roundings of the parts and one of the result, on both sides
    size = float(case.v.float().abs().max())
    assert float((merged.float() - whole.float()).abs().max()) <= 4 * 2.0**-11 * size
    assert float((lse - whole_lse).abs().max()) <= 1e-3


def test_repeat_graph_and_operator():
    case = Case([300, 700, 64], [400, 700, 1000], 4, seed=23)
    first = tsb.latent_prompt_attention(*case.args())
    for _ in range(10):
        assert torch.equal(tsb.latent_prompt_attention(*case.args()), first)
    assert torch.equal(torch.ops.b200kv.latent_prompt_attention(*case.args(), 192**-0.5, True, None)[0], first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tsb.latent_prompt_attention(*case.args())
    captured.zero_()
    graph.replay()
    assert torch.equal(captured, first)


def test_a_graph_follows_the_offsets():
    # the plan is made on the device: other prompts of the same numbers of rows and tokens in all
    case = Case([300, 700, 64], [400, 700, 1000], 4, seed=24)
    tsb.latent_prompt_attention(*case.args())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tsb.latent_prompt_attention(*case.args())
    for q_ptr, kv_ptr in (((0, 1, 1000, 1064), (0, 1, 1900, 2100)), ((0, 0, 1064, 1064), (0, 500, 2000, 2100)),
                          ((0, 400, 500, 1064), (0, 300, 600, 2100))):
        case.q_indptr.copy_(torch.tensor(q_ptr, dtype=torch.int32))
        case.kv_indptr.copy_(torch.tensor(kv_ptr, dtype=torch.int32))
        graph.replay()
        assert torch.equal(captured, tsb.latent_prompt_attention(*case.args()))


@pytest.mark.parametrize("heads", [37, 100])
def test_many_short_blocks_to_a_share(heads):
    # blocks of one and two Q tiles, with warps that have no row, one after the other on every SM
    new = [1, 70, 33, 129, 161, 300, 44, 257, 96, 5]
    check(Case(new, [n + p for n, p in zip(new, [0, 79, 80, 0, 33, 1, 500, 7, 160, 81])], heads, seed=heads))
