"""The drafting example at the end of its context."""
import pytest
import torch

import test_gpu_drafting  # noqa: F401  (finds the example)
import draft_four_models as ex

pytestmark = pytest.mark.gpu


def test_texts_end_with_the_context():
    """Every step that the context has room for, to its last token; no step beyond it, and no prompt beyond it."""
    g = torch.Generator().manual_seed(5)
    models = ex.Drafting(context=40, drafts=3)
    models.begin(torch.randint(0, ex.VOCAB, (ex.MODELS, 32), generator=g).cuda())
    for _ in range(3):                                            # texts of up to 32, 36 and 40 tokens before them
        models.step(torch.rand(ex.MODELS, 4, generator=g).cuda())
    sizes = models.size.tolist()
    with pytest.raises(ValueError, match="context"):
        models.step(torch.rand(ex.MODELS, 4, generator=g).cuda())
    assert models.size.tolist() == sizes and max(sizes) <= 44
    with pytest.raises(ValueError, match="context"):
        models.begin(torch.zeros(ex.MODELS, 41, dtype=torch.int64).cuda())
