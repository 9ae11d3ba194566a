"""Four packed models continue their texts several tokens a step: drafts looked up in the text itself, checked against
each model's own probabilities; rotary positions, and a cache in 4 bits.

    python -m examples.draft_four_models       (from the root of the repository)

The models are those of :mod:`decode_four_models`.  A step feeds each model its last token and the drafts after it, which
join the cache; the tokens it keeps stay there, and what lies behind them is written over by the next step.  Lengths
differ from model to model and stay on the device: nothing here waits for it.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from decode_four_models import BLOCK, HEAD, KV_HEADS, MODELS, Q_HEADS, VOCAB, Models  # noqa: E402

from polar_pack_amd.drafts import verify_drafts  # noqa: E402
from polar_pack_amd.kv_cache import KVCache4, kv_attention, kv_rotate_append  # noqa: E402
from polar_pack_amd.rotary import Rotary  # noqa: E402


class Drafting(Models):
    """The four models with positions, their caches in 4 bits and their texts."""

    def __init__(self, device="cuda", context=256, drafts=4):
        super().__init__(device, context=BLOCK)
        pages = -(-(context + drafts) // BLOCK)
        self.cache = KVCache4.zeros(MODELS * pages, KV_HEADS, HEAD, block=BLOCK, device=device)
        self.table = torch.arange(MODELS * pages, dtype=torch.int32, device=device).view(MODELS, pages)
        self.rotary = Rotary(HEAD, device=device)
        self.drafts = drafts
        self.text = torch.zeros(MODELS, context + drafts + 1, dtype=torch.int64, device=device)
        self.size = torch.zeros(MODELS, dtype=torch.int64, device=device)
        self.context, self.most = context, 0

    def forward(self, tokens, lengths):
        """Logits (models, n, VOCAB) after each of ``tokens`` (models, n), the last of ``lengths`` (models,) each."""
        n = tokens.shape[1]
        x = self.embed[torch.arange(MODELS, device=tokens.device)[:, None], tokens]
        qkv = self.linear(0, x).view(MODELS * n, Q_HEADS + 2 * KV_HEADS, HEAD)
        q, k, v = qkv.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        at = (self.table, lengths.int(), torch.arange(MODELS + 1, dtype=torch.int32, device=tokens.device) * n)
        q = kv_rotate_append(self.cache, q, k, v, self.rotary, *at)
        heads = kv_attention(q, self.cache, *at)
        return self.linear(2, x + self.linear(1, heads.view(MODELS, n, Q_HEADS * HEAD)))

    def begin(self, prompt):
        """Take in all of ``prompt`` (models, n) but its last token."""
        n = prompt.shape[1]
        if n > self.context:
            raise ValueError(f"a prompt of {n} tokens in a context of {self.context}")
        self.text[:, :n] = prompt
        self.most = n
        self.size.fill_(n)
        self.forward(prompt[:, :-1], self.size - 1)

    def look_up(self):
        """The tokens that followed the last earlier occurrence of a text's last token, and how many there are."""
        place = torch.arange(self.text.shape[1], device=self.text.device)
        last = self.text.gather(1, self.size[:, None] - 1)
        found = (self.text == last) & (place < self.size[:, None] - 1)
        at = torch.where(found, place, -1).amax(1)
        tokens = self.text.gather(1, (at[:, None] + 1 + place[:self.drafts]).clamp(0, self.text.shape[1] - 1))
        counts = torch.where(at < 0, 0, (self.size - 1 - at).clamp(max=self.drafts))
        return last, tokens, counts.int()

    def step(self, uniforms, temperature=0.7):
        """One step with ``uniforms`` (models, drafts + 1): what was drafted and what became of it.  How long the texts are
        only the device knows, so a step is refused where they could be longer than the context, all drafts kept."""
        if self.most > self.context:
            raise ValueError(f"texts of up to {self.most} tokens in a context of {self.context}")
        self.most += self.drafts + 1
        last, tokens, counts = self.look_up()
        logits = self.forward(torch.cat([last, tokens], 1), self.size + self.drafts)
        target = torch.softmax(logits.float() / temperature, 2)
        r = verify_drafts(target, None, tokens, uniforms, counts)
        at = self.size[:, None] + torch.arange(self.drafts + 1, device=self.text.device)
        self.text.scatter_(1, at, r.tokens.clamp(min=0))
        self.size += r.accepted + 1
        return target, tokens, counts, r


if __name__ == "__main__":
    models = Drafting()
    g = torch.Generator().manual_seed(1)
    phrase = torch.randint(0, VOCAB, (MODELS, 20), generator=g)
    models.begin(torch.cat([phrase, phrase], 1).cuda())
    kept = torch.stack([models.step(torch.rand(MODELS, models.drafts + 1, generator=g).cuda())[3].accepted for _ in range(8)])
    for m, (size, accepted) in enumerate(zip(models.size.tolist(), kept.t().tolist())):
        print(f"model {m}: {models.text[m, 40:size].tolist()}, drafts kept {accepted}")
