"""token_logprobs against log_softmax in 64 bits.

The bounds: exp of a float32 difference d is off by a relative |d| 2^-24 plus 2^-22, so the sum by 2^-19
at the differences that count (|d| <= 40; smaller terms weigh e^-40), and sums of float32 partial sums
add about 2^-20; a result is rounded at its magnitude (2^-23 of |x| + |lse|)."""
import math

import pytest
import torch

from polar_pack_amd.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def check(x, tokens, top):
    r = token_logprobs(x.to(DEV) if x.device.type == "cpu" else x, tokens.to(DEV), top=top)
    x = x.cpu()
    lp = torch.log_softmax(x.double(), 1)
    V = x.shape[1]
    tk = tokens if tokens.dim() == 2 else tokens[:, None]
    ok = (tk >= 0) & (tk < V)
    want = torch.where(ok, lp.gather(1, tk.clamp(0, V - 1)), math.nan).view(tokens.shape)
    big = x.double().nan_to_num(0, 0, 0).abs().amax(1)
    tol = 2.0 ** -18 + 2.0 ** -22 * (big + math.log(V))

    def near(got, want, tol, what):
        got = got.cpu().double()
        good = (got == want) | (got.isnan() & want.isnan()) | ((got - want).abs() <= tol)
        assert good.all(), (what, (got - want).abs().nan_to_num(0, 0, 0).max(), good.logical_not().nonzero()[:3])
    near(r.logprob, want, tol if tokens.dim() == 1 else tol[:, None], "logprob")
    ent = -torch.where(lp == -math.inf, 0.0, lp.exp() * lp).sum(1)
    near(r.entropy, ent, tol * (2 + ent.nan_to_num(0)), "entropy")
    if top:
        order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids.cpu(), order), (r.top_ids.cpu() != order).nonzero()[:5]
        near(r.top_logprobs, lp.gather(1, order), tol[:, None], "alternatives")
    else:
        assert r.top_ids is None and r.top_logprobs is None
    return r


def logits(rows, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * spread).to(dtype)
    return x, torch.randint(0, V, (rows,), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 63), (5, 4096), (1, 4097), (4, 50001), (1, 151936), (600, 1003)])
def test_matches_64_bits(rows, V, dtype):
    for top in sorted({0, 1, min(5, V), min(64, V)}):
        check(*logits(rows, V, dtype, rows + V), top)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_as_long_as_a_workgroup_walks(dtype):
    """Enough rows that each is one workgroup's: its list is shortened as it walks."""
    check(*logits(520, 20011, dtype, 3), 20)


@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("rows", [1, 520])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two", "steps", "masked"])
def test_orders_and_ties(kind, rows, top):
    """Orders that hit the list hardest: every logit above all before, every logit equal, few values."""
    V = 17001
    i = torch.arange(V).float()
    x = {"equal": torch.zeros(V), "rising": i / 1000, "falling": -i / 1000, "two": (i % 2), "steps": (i // 700) % 7,
         "masked": torch.where(i % 400 == 3, i / 9000, -math.inf)}[kind]
    check(x[None].repeat(rows, 1), torch.arange(rows) * 7 % V, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
    V = 9001
    x, t = logits(7, V, dtype, 5)
    x[0, ::2] = -math.inf
    x[1] = -math.inf                                # nothing left
    x[2, 17] = math.nan
    x[3, 8000] = math.inf
    x[4, :] = torch.finfo(dtype).min
    x[5, 1:] = -math.inf                            # one logit left
    x[6, 4] = torch.finfo(dtype).max
    t[5] = 0
    r = check(x, t, 4)
    assert r.logprob[5] == 0 and r.entropy[5] == 0
    assert r.logprob[1:4].isnan().all() and r.top_ids[2, 0] == 17 and r.top_ids[3, 0] == 8000
    check(torch.tensor([[-0.0, 0.0, -0.0, 0.0]]), torch.tensor([1]), 4)      # equal: the lower index


def test_several_tokens_a_row_and_tokens_out_of_range():
    x, _ = logits(3, 5000, torch.float16, 2)
    g = torch.Generator().manual_seed(1)
    t = torch.randint(0, 5000, (3, 300), generator=g)
    t[0, 0], t[1, 5], t[2, 2] = -1, 5000, 2 ** 40
    r = check(x, t, 3)
    assert r.logprob[0, 0].isnan() and r.logprob[1, 5].isnan() and r.logprob[2, 2].isnan()
    check(x, t[:, :0], 3)
    check(x, t[:, ::2], 0)
    check(x, t.t().contiguous().t(), 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    x, t = logits(6, 5003, dtype, 4)
    for pad, off in ((0, 0), (1, 1), (5, 3), (8, 8)):
        wide = torch.full((6, 5003 + pad), 99.0, dtype=dtype, device=DEV)
        part = wide[:, off:off + 5003]
        part.copy_(x)
        check(part, t, 5)
    check(x.to(DEV)[::2], t[::2], 5)
    check(x[:1].to(DEV).expand(6, 5003), t, 5)
    check(x.t().contiguous().to(DEV).t(), t, 5)


def test_logits_that_negate_when_they_are_read():
    for dtype in (torch.float16, torch.float32):
        x, t = logits(5, 3001, dtype, 6)
        x = x.to(DEV)
        view = torch._neg_view(-x)
        assert view.is_neg() and torch.equal(view, x)
        check(view, t, 3)
        for a, b in zip(token_logprobs(view, t.to(DEV), top=3), token_logprobs(x, t.to(DEV), top=3)):
            assert torch.equal(a, b)


def test_no_rows():
    r = token_logprobs(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), top=3)
    assert r.logprob.shape == (0,) and r.entropy.shape == (0,) and r.top_ids.shape == (0, 3)


@pytest.mark.parametrize("rows", [2, 520])
def test_in_a_graph_and_on_another_stream(rows):
    x, t = logits(rows, 30000, torch.float16, 8)
    x, t = x.to(DEV), t.to(DEV)
    want = token_logprobs(x, t, top=7)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = token_logprobs(x, t, top=7)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, t, top=7)
    for a, b in zip(other, want):
        assert torch.equal(a, b)
    for i in range(3):
        x.copy_(x.roll(i + 1, 1))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, token_logprobs(x, t, top=7)):
            assert torch.equal(a, b), i


def test_refusals():
    x = torch.zeros(2, 10, device=DEV)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError):
        token_logprobs(x.double(), t)
    with pytest.raises(TypeError):
        token_logprobs(x, t.int())
    with pytest.raises(TypeError):
        token_logprobs(x, t[:1])
    with pytest.raises(ValueError):
        token_logprobs(x, t, top=11)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(2, 100, device=DEV), t, top=65)
    with pytest.raises(ValueError):
        token_logprobs(x, t, top=-1)
    with pytest.raises(ValueError):
        token_logprobs(x.cpu(), t)
    with pytest.raises(ValueError):
        token_logprobs(x[:, :0], t)
