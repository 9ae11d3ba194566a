"""verify_drafts against its definition in 64 bits, a sequence at a time: whole numbers, so equal ones.

Sums of at most 2^18 entries in 64 bits are off by less than 2^-35 of the whole whatever their order, and a number u of
24 bits lies that near to one of the sums' steps by chance once in some 10^5 rows of this length, of which a few thousand
are drawn here at most from the longest; the cases are fixed."""
import math

import pytest
import torch

from polar_pack_amd.drafts import verify_drafts
from serving import DEV

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def clean(x):
    return x.double().nan_to_num(0.0).clamp(0.0, torch.finfo(torch.float32).max)


def plain(p, q, tokens, u, counts=None):
    B, n = tokens.shape
    V = p.shape[2]
    out, accepted = torch.full((B, n + 1), -1), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        c = n if counts is None else min(max(int(counts[b]), 0), n)
        i = 0
        while i < c:
            d = int(tokens[b, i])
            known = 0 <= d < V
            pd = float(clean(p[b, i, d])) if known else 0.0
            qd = 1.0 if q is None else float(clean(q[b, i, d])) if known else 0.0
            if not float(u[b, i]) * qd < pd:
                break
            out[b, i] = d
            i += 1
        row = clean(p[b, i])
        rest = row
        if i < c:
            if q is None:
                rest = row.clone()
                if 0 <= int(tokens[b, i]) < V:
                    rest[int(tokens[b, i])] = 0
            else:
                rest = (row - clean(q[b, i])).clamp(min=0)
        if not rest.sum() > 0:
            rest = row
        total = rest.cumsum(0)
        if total[-1] > 0:
            past = total > max(float(u[b, n]), 0.0) * total[-1]
            out[b, i] = int(past.int().argmax()) if past.any() else int((rest > 0).nonzero()[-1])
        accepted[b] = i
    return out, accepted


def problem(B, n, V, dtype, seed, sharp=2.0, near=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, n + 1, V, generator=g) * sharp
    p = torch.softmax(x, 2).to(dtype)
    d = torch.softmax(x[:, :n] + near * torch.randn(B, n, V, generator=g), 2)
    tokens = torch.multinomial(d.flatten(0, 1), 1, generator=g).view(B, n) if n else torch.empty(B, 0, dtype=torch.int64)
    return p, d.to(dtype), tokens, torch.rand(B, n + 1, generator=g)


def check(p, q, tokens, u, counts=None):
    got = verify_drafts(*(t if t is None else t.to(DEV) for t in (p, q, tokens, u, counts)))
    want = plain(p, q, tokens, u, counts)
    assert torch.equal(got.accepted.cpu(), want[1])
    assert torch.equal(got.tokens.cpu(), want[0])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 255, 1000, 4095, 4096, 4097, 8195, 30001])
def test_vocabularies(V, draft, dtype):
    p, q, tokens, u = problem(9, 3, V, dtype, V)
    check(p, q if draft else None, tokens, u)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_vocabulary(dtype):
    p, q, tokens, u = problem(4, 4, 151936, dtype, 1)
    check(p, q, tokens, u)
    check(p, None, tokens, u)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("B,n", [(1, 1), (1, 0), (300, 0), (2, 63), (2, 64), (3, 65), (2, 200), (700, 2)])
def test_batches_and_drafts(B, n, draft):
    """None, few, more than a wavefront looks at; near to the target, so that many are kept."""
    p, q, tokens, u = problem(B, n, 300, torch.float32, B + n, near=0.02)
    got = check(p, q if draft else None, tokens, u)
    if draft and n > 60:
        assert int(got.accepted.max()) > 10


@pytest.mark.parametrize("B", [1, 40, 3000])
def test_parts_of_a_row(B):
    """Rows cut into many parts, few, none: one case of each, tokens from everywhere in the row."""
    V = 70001 if B == 1 else 20003 if B == 40 else 500
    p, q, tokens, u = problem(B, 1, V, torch.float32, B, sharp=0.3)
    got = check(p, q, tokens, u)
    if B == 40:
        assert int(got.tokens.max()) > 15000


@pytest.mark.parametrize("draft", [True, False])
def test_counts(draft):
    """Fewer drafts than places, none, more than there are, below zero; what lies past them is not read."""
    p, q, tokens, u = problem(8, 5, 100, torch.float32, 3, near=0.1)
    counts = torch.tensor([0, 1, 2, 3, 4, 5, 9, -2], dtype=torch.int32)
    want = plain(p, q if draft else None, tokens, u, counts)
    for b, c in enumerate(counts.clamp(0, 5).tolist()):
        p[b, c + 1:], q[b, c:], tokens[b, c:], u[b, c:5] = math.nan, math.nan, -9, math.nan
    got = check(p, q if draft else None, tokens, u, counts)
    assert torch.equal(got.tokens.cpu(), want[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("u_last", [0.0, 0.5, 1 - 2.0 ** -24, 1.0, 1.5, -1.0])
def test_the_ends_of_a_row(u_last, dtype):
    """Zeros before, between and behind; the first and the last that are not; numbers outside [0, 1)."""
    p = torch.zeros(3, 1, 9001, dtype=dtype)
    p[0, 0, 4], p[0, 0, 8990] = 0.5, 0.5
    p[1, 0, 9000] = 2.0 ** -14
    p[2, 0, 5000:5004] = 0.25
    u = torch.full((3, 1), u_last)
    got = check(p, None, torch.empty(3, 0, dtype=torch.int64), u)
    if u_last <= 0:
        assert got.tokens[:, 0].tolist() == [4, 9000, 5000]
    if u_last >= 1:
        assert got.tokens[:, 0].tolist() == [8990, 9000, 5003]


def test_acceptance_at_its_border():
    """u q < p, not <=; a token the target never says is refused even at u = 0; one it is sure of is kept."""
    p = torch.zeros(4, 2, 4)
    q = torch.zeros(4, 1, 4)
    p[:, :, 3] = 1.0
    p[0, 0, 1], q[0, 0, 1] = 0.25, 0.5
    p[1, 0, 1], q[1, 0, 1] = 0.25, 0.5
    q[2, 0, 1] = 0.5
    p[3, 0, 1], q[3, 0, 1] = 0.25, 0.0
    tokens, u = torch.ones(4, 1, dtype=torch.int64), torch.tensor([[0.5, 0.5], [0.49999997, 0.5], [0.0, 0.5], [0.999, 0.5]])
    got = check(p, q, tokens, u)
    assert got.accepted.tolist() == [0, 1, 0, 1]


def test_nothing_left():
    """p at or below q everywhere: the token is p's; rows of nothing give -1."""
    p = torch.zeros(4, 2, 5000)
    p[:3, 0, 100:110] = 0.1
    q = torch.full((4, 1, 5000), 1.0)
    tokens, u = torch.full((4, 1), 7), torch.full((4, 2), 0.35)
    got = check(p, q, tokens, u)
    assert got.accepted.tolist() == [0] * 4 and got.tokens[:, 0].tolist() == [103, 103, 103, -1]
    one = torch.zeros(1, 2, 5000)
    one[0, 0, 7] = 1e-9
    got = check(one, None, tokens[:1], torch.full((1, 2), 0.5))          # refused, and nothing else there
    assert got.tokens.tolist() == [[7, -1]]


@pytest.mark.parametrize("dtype", TYPES)
def test_entries_that_are_no_probabilities(dtype):
    p, q, tokens, u = problem(6, 2, 600, dtype, 5)
    for x in (p, q):
        x[0, :, 3::7], x[1, :, 4::5], x[2, :, ::3], x[3] = math.nan, math.inf, -1.0, math.nan
    tokens[4, 0], tokens[5, 0] = -1, 600
    check(p, q, tokens, u)
    check(p, None, tokens, u)


def test_rows_need_not_add_up_to_one():
    p, q, tokens, u = problem(20, 2, 1000, torch.float32, 6)
    check(p * 1e30, q * 1e30, tokens, u)
    check(p * 1e-30, q * 1e-30, tokens, u)


def test_places_and_strides():
    p, q, tokens, u = problem(5, 3, 333, torch.float32, 7)
    want = plain(p, q, tokens, u)
    P, Q, T, U = (t.to(DEV) for t in (p, q, tokens, u))
    wide = torch.full((5, 4, 400), math.nan, device=DEV)
    wide[:, :, 61:394] = P
    forms = [(wide[:, :, 61:394], Q, T, U), (P.transpose(0, 1).contiguous().transpose(0, 1), Q, T, U),
             (P.transpose(1, 2).contiguous().transpose(1, 2), Q.transpose(0, 2).contiguous().transpose(0, 2), T, U),
             (torch._neg_view(-P), torch._neg_view(-Q), T, torch._neg_view(-U)),
             (P, Q, T.t().contiguous().t(), U.t().contiguous().t()),
             (P, Q, torch.stack([T, T], 2)[:, :, 0], torch.cat([U, U], 1)[:, :4])]
    for args in forms:
        got = verify_drafts(*args)
        assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])
    same = verify_drafts(P[:1].expand(5, 4, 333), Q[:1].expand(5, 3, 333), T[:1].expand(5, 3), U)
    assert torch.equal(same.tokens.cpu(), plain(*(t[:1].expand(5, *t.shape[1:]) for t in (p, q, tokens)), u)[0])


def test_the_answer_is_distributed_as_the_target():
    """The first token of 200,000 draws: frequencies within 6 standard deviations of the target's row."""
    B, V = 200_000, 8
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, V, generator=g)
    p, q = torch.softmax(x, 1), torch.softmax(x[:1] + torch.randn(1, V, generator=g), 1)
    tokens = torch.multinomial(q[0], B, replacement=True, generator=g)[:, None]
    u = torch.rand(B, 2, generator=g)
    got = verify_drafts(p.to(DEV).expand(B, 2, V), q.to(DEV).expand(B, 1, V), tokens.to(DEV), u.to(DEV))
    share = torch.bincount(got.tokens[:, 0].cpu(), minlength=V) / B
    assert ((share - p[0]).abs() <= 6 * (p[0] * (1 - p[0]) / B).sqrt()).all()
    kept = torch.minimum(p[0], q[0]).sum()
    assert (got.accepted.double().mean().cpu() - kept).abs() <= 6 * (kept * (1 - kept) / B).sqrt()


def test_capture_and_streams():
    """Replayed with new numbers between eager calls on the same and on another stream; the counts are left zero."""
    p, q, tokens, u = (t.to(DEV) for t in problem(6, 3, 20000, torch.float32, 10))
    verify_drafts(p, q, tokens, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = verify_drafts(p, q, tokens, u)
    side = torch.cuda.Stream()
    for step in range(5):
        p.copy_(torch.softmax(torch.randn_like(p) * 2, 2))
        u.uniform_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = verify_drafts(p, q, tokens, u)
        torch.cuda.current_stream().wait_stream(side)
        r.tokens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.tokens, want.tokens) and torch.equal(r.accepted, want.accepted)
        again = verify_drafts(p, q, tokens, u)
        assert torch.equal(again.tokens, want.tokens)


def test_nothing_to_check():
    r = verify_drafts(torch.empty(0, 3, 10, device=DEV), None, torch.empty(0, 2, dtype=torch.int64, device=DEV),
                      torch.empty(0, 3, device=DEV))
    assert r.tokens.shape == (0, 3) and r.accepted.shape == (0,)


def test_refusals():
    p, q, tokens, u = (t.to(DEV) for t in problem(2, 3, 50, torch.float32, 11))
    counts = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    for bad, exc in ((lambda: verify_drafts(p.double(), q, tokens, u), TypeError), (lambda: verify_drafts(p[0], q, tokens, u), TypeError),
                     (lambda: verify_drafts(p[:, :0], q[:, :0], tokens[:, :0], u), ValueError),
                     (lambda: verify_drafts(p, q.half(), tokens, u), ValueError), (lambda: verify_drafts(p, q[:, :2], tokens, u), ValueError),
                     (lambda: verify_drafts(p, q, tokens.int(), u), TypeError), (lambda: verify_drafts(p, q, tokens[:, :2], u), TypeError),
                     (lambda: verify_drafts(p, q, tokens, u[:, :3]), TypeError), (lambda: verify_drafts(p, q, tokens, u.double()), TypeError),
                     (lambda: verify_drafts(p, q, tokens, u, counts.long()), TypeError), (lambda: verify_drafts(p, q, tokens, u, counts[:1]), TypeError),
                     (lambda: verify_drafts(p[..., :0], q[..., :0], tokens, u), ValueError),
                     (lambda: verify_drafts(p, q.cpu(), tokens, u), ValueError), (lambda: verify_drafts(p.cpu(), None, tokens.cpu(), u.cpu()), ValueError)):
        with pytest.raises(exc):
            bad()
