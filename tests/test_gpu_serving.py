"""The serving operators together, as the example runs them: packed Linears, cache, attention, answers."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import decode_four_models as ex  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_prompt_and_single_tokens_agree(codes):
    """The logits after a prompt taken in at once and token by token.  Both see the same queries; keys and
    values differ by how often a page's codes were rounded as its scale grew: a step of 1/127 of a page's
    largest value (e4m3: a relative 1/16) a time, a few times a page of 64 tokens, spread over all of them."""
    prompt = torch.randint(0, ex.VOCAB, (ex.MODELS, 70), generator=torch.Generator().manual_seed(1)).cuda()
    whole = ex.Models(codes=codes).forward(prompt)
    models = ex.Models(codes=codes)
    for i in range(prompt.shape[1]):
        last = models.forward(prompt[:, i:i + 1])
    scale = whole.float().std()
    assert torch.isfinite(whole).all()
    assert (whole.float() - last.float()).abs().max() < (0.05 if codes == torch.int8 else 0.25) * scale


def test_answers():
    prompt = torch.randint(0, ex.VOCAB, (ex.MODELS, 40), generator=torch.Generator().manual_seed(1)).cuda()
    tokens, logprob, entropy, top = ex.answer(ex.Models(), prompt, 4)
    assert torch.equal(tokens, top[..., 0])            # greedy: the chosen token is the first alternative
    assert (logprob <= 0).all() and (entropy > 0).all() and (entropy < 7).all()      # ln 1000 = 6.9
    assert len({tuple(t) for t in tokens.tolist()}) > 1                              # four models, not one
