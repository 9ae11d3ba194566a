"""Four packed models answer a prompt in lock step: packed Linears, the 8-bit cache, its attention and
the log probabilities of what is chosen.

    python -m examples.decode_four_models       (from the root of the repository)

A one-layer decoder of random weights stands for each model.  Its Linears come from one
quad stream; the four models' rows go through a Linear together, each keeping its own model's
output.  Their sequences are four rows of one block table, so one launch appends to, and one
attends to, all four caches.
"""
import torch

from polar_pack_amd.kv_cache import KVCache, kv_append, kv_attention
from polar_pack_amd.linear import QuadPackedLinear
from polar_pack_amd.logprobs import token_logprobs
from polar_pack_amd.packer import pack_quad_device

MODELS, WIDTH, Q_HEADS, KV_HEADS, HEAD, VOCAB, BLOCK = 4, 512, 8, 2, 64, 1000, 64
SHAPES = [((Q_HEADS + 2 * KV_HEADS) * HEAD, WIDTH), (WIDTH, Q_HEADS * HEAD), (VOCAB, WIDTH)]


class Models:
    """The packed weights, the embeddings and the caches of four decoders."""

    def __init__(self, device="cuda", codes=torch.int8, context=256):
        g = torch.Generator().manual_seed(0)
        base = [torch.randn(s, generator=g) * s[1] ** -0.5 for s in SHAPES]
        weights = [[(w + 0.2 * torch.randn(w.shape, generator=g) * w.std()).half().to(device) for w in base]
                   for _ in range(MODELS)]
        pack = pack_quad_device(weights)
        self.linears, at = [], 0
        for n, k in SHAPES:
            self.linears.append(QuadPackedLinear(pack, n, k, at))
            at += n * k
        self.embed = torch.randn(MODELS, VOCAB, WIDTH, generator=g).half().to(device)
        pages = -(-context // BLOCK)
        self.cache = KVCache.zeros(MODELS * pages, KV_HEADS, HEAD, block=BLOCK, dtype=codes, device=device)
        self.table = torch.arange(MODELS * pages, dtype=torch.int32, device=device).view(MODELS, pages)
        self.length = 0

    def linear(self, i, x):
        """(models, tokens, K) -> (models, tokens, N): every model's rows through its own weights."""
        m, t, k = x.shape
        ys = self.linears[i](x.reshape(m * t, k))
        return torch.stack([y.view(m, t, -1)[j] for j, y in enumerate(ys)])

    def forward(self, tokens):
        """Logits (models, VOCAB) after ``tokens`` (models, n), which join the caches."""
        n = tokens.shape[1]
        self.length += n
        x = self.embed[torch.arange(MODELS, device=tokens.device)[:, None], tokens]
        qkv = self.linear(0, x).view(MODELS * n, Q_HEADS + 2 * KV_HEADS, HEAD)
        q, k, v = qkv.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        lengths = torch.full((MODELS,), self.length, dtype=torch.int32, device=tokens.device)
        cu = None if n == 1 else torch.arange(MODELS + 1, dtype=torch.int32, device=tokens.device) * n
        kv_append(self.cache, k, v, self.table, lengths, cu)
        heads = kv_attention(q, self.cache, self.table, lengths, cu)
        x = x + self.linear(1, heads.view(MODELS, n, Q_HEADS * HEAD))
        return self.linear(2, x[:, -1:])[:, 0]


def answer(models, prompt, steps, top=3):
    """Greedy tokens (models, steps), their log probabilities, the entropies and the alternatives."""
    logits, out = models.forward(prompt), []
    for _ in range(steps):
        chosen = logits.argmax(1)
        out.append((chosen, token_logprobs(logits, chosen, top=top)))
        logits = models.forward(chosen[:, None])
    return (torch.stack([c for c, _ in out], 1), torch.stack([r.logprob for _, r in out], 1),
            torch.stack([r.entropy for _, r in out], 1), torch.stack([r.top_ids for _, r in out], 1))


if __name__ == "__main__":
    models = Models()
    prompt = torch.randint(0, VOCAB, (MODELS, 40), generator=torch.Generator().manual_seed(1)).cuda()
    tokens, logprob, entropy, alternatives = answer(models, prompt, 8)
    for m in range(MODELS):
        print(f"model {m}: " + " ".join(f"{t}({p:.2f})" for t, p in zip(tokens[m].tolist(), logprob[m].tolist()))
              + f"  mean entropy {entropy[m].mean():.2f}, alternatives of the first {alternatives[m, 0].tolist()}")
