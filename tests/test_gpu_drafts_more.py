"""verify_drafts where the first tests of it do not look: counts beside the 64 drafts that a wavefront looks at."""
import pytest
import torch

from test_gpu_drafts import check, plain, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draft", [True, False])
def test_counts_of_many_drafts(draft):
    """None, one, and either side of whole rounds of 64; the numbers are such that most drafts are kept, so counts end them.
    What lies past them is NaN, or no token of the vocabulary."""
    counts = torch.tensor([0, 1, 63, 64, 65, 127, 128, 129, 130], dtype=torch.int32)
    p, q, tokens, u = problem(9, 130, 100, torch.float32, 5, near=0.001)
    u[:, :130] *= 0.001
    q = q if draft else None
    want = plain(p, q, tokens, u, counts)
    if draft:
        assert int((want[1] == counts).sum()) >= 6
    for b, c in enumerate(counts.tolist()):
        p[b, c + 1:], tokens[b, c:], u[b, c:130] = float("nan"), -9, float("nan")
        if draft:
            q[b, c:] = float("nan")
    got = check(p, q, tokens, u, counts)
    assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])
