"""Rotary positions, the 4-bit cache, its attention and the check of drafts together, as the example runs them."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import draft_four_models as ex  # noqa: E402
from test_gpu_drafts import plain  # noqa: E402

pytestmark = pytest.mark.gpu


def start(drafts=4):
    phrase = torch.randint(0, ex.VOCAB, (ex.MODELS, 12), generator=torch.Generator().manual_seed(1))
    models = ex.Drafting(drafts=drafts)
    models.begin(torch.cat([phrase, phrase], 1).cuda())
    return models


def test_steps_do_what_the_definition_says():
    """Every step's tokens against the plain check of the same probabilities, drafts and numbers; texts grow by them."""
    models, g = start(), torch.Generator().manual_seed(2)
    grown, kept = [[] for _ in range(ex.MODELS)], 0
    for i in range(6):
        before = models.size.clone()
        u = torch.rand(ex.MODELS, models.drafts + 1, generator=g)
        if i % 2 == 0:                                       # at first, while the text repeats itself
            u[:, 1:-1] = 0                                    # what has a probability at all is kept
            u[::2, 0] = 0
        target, tokens, counts, r = models.step(u.cuda())
        want, accepted = plain(target.cpu(), None, tokens.cpu(), u, counts.cpu())
        assert torch.equal(r.tokens.cpu(), want) and torch.equal(r.accepted.cpu(), accepted)
        assert torch.equal((models.size - before).cpu(), accepted + 1)
        kept += int(accepted.sum())
        for m in range(ex.MODELS):
            grown[m] += [t for t in want[m].tolist() if t >= 0]
    for m in range(ex.MODELS):
        assert models.text[m, 24:int(models.size[m])].tolist() == grown[m]
    assert kept > 0


def test_drafts_that_were_refused_leave_nothing_behind():
    """The probabilities after some steps, refused drafts among them, and after the same texts at once.  Both see the same
    tokens; a key or value differs where its 16-bit inputs, from products of other row counts, were rounded to the other side of a
    code's border: few of them, by one step of a group of 32, a seventh to a quarter of its largest, so that logits move by a small
    part of their spread (one value in a hundred by a step in 64 terms of unit size: below a quarter of it)."""
    models, g = start(), torch.Generator().manual_seed(3)
    for i in range(5):
        u = torch.rand(ex.MODELS, models.drafts + 1, generator=g)
        if i % 2 == 0:                                       # at first, while the text repeats itself
            u[:, :2] = 0
        models.step(u.cuda())
    last = models.text.gather(1, models.size[:, None] - 1)
    stepped = models.forward(last, models.size)[:, 0].float()
    for m in range(ex.MODELS):
        n = int(models.size[m])
        fresh = ex.Drafting()
        whole = fresh.forward(models.text[:, :n], torch.full((ex.MODELS,), n, device="cuda"))[m, -1].float()
        assert torch.isfinite(whole).all()
        assert (whole - stepped[m]).abs().max() < 0.25 * whole.std()


def test_without_drafts_a_step_is_a_token():
    models = start(drafts=1)
    models.look_up = lambda: (models.text.gather(1, models.size[:, None] - 1),
                              torch.zeros(ex.MODELS, 1, dtype=torch.int64, device="cuda"),
                              torch.zeros(ex.MODELS, dtype=torch.int32, device="cuda"))
    for _ in range(3):
        before = models.size.clone()
        r = models.step(torch.full((ex.MODELS, 2), 0.5, device="cuda"))[3]
        assert torch.equal(models.size, before + 1) and (r.tokens[:, 1] == -1).all() and (r.tokens[:, 0] >= 0).all()


def test_a_step_in_a_graph():
    """Captured once and replayed with new numbers, beside the same steps run eagerly."""
    one, two, g = start(), start(), torch.Generator().manual_seed(4)
    u = torch.rand(ex.MODELS, one.drafts + 1, generator=g).cuda()
    for models in (one, two):
        models.step(u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = two.step(u)[3]
    for _ in range(4):
        u.copy_(torch.rand(ex.MODELS, one.drafts + 1, generator=g))
        want = one.step(u)[3]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.tokens, want.tokens) and torch.equal(one.size, two.size) and torch.equal(one.text, two.text)
