"""kv_attention over the 4-bit cache where the first tests of it do not look: large values behind tiny weights."""
import math

import pytest
import torch

from polar_pack_amd.kv_cache import kv_attention
from serving import DEV, attention, offsets
from serving4 import device_cache4, plain_parts, random_cache4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("many", [1, 12, 150])
@pytest.mark.parametrize("nats", [12, 20, 25, 28, 32])
@pytest.mark.parametrize("top,rest", [(-14, 13), (-14, 0), (0, 13)])
def test_large_values_behind_tiny_weights(top, rest, nats, many):
    """One key ahead of 299 by so many nats, whose values have a scale of 2^rest where its own have 2^top.  Weights of 11 bits
    (in serving.attention's bound), or within 2^-39 of the largest (4 to 48 rows; 600 rows: 2^-37), times their values.  Outputs in
    fp16, the smallest of them held to half a step of 2^-24 (in the bound's 1e-7)."""
    L, D = 300, 64
    g = torch.Generator().manual_seed(nats)
    parts = random_cache4(5, 1, 64, D, g, 0, 1)
    parts[0].fill_(0xaa)                                     # codes -1, and 1 at one key
    parts[0][1, 0, 6] = 0x22
    table = torch.arange(5, dtype=torch.int32)[None]
    vs = torch.full((5, 1, D // 32, 64), 2.0 ** rest)
    vs[1, 0, :, 6] = 2.0 ** top
    parts = (*parts[:3], vs.to(torch.float8_e5m2))
    q, scale = torch.ones(many, 4, D, dtype=torch.float16), nats / 128
    want, lse, tol, tol_lse = attention(q, plain_parts(parts), table, [L], [many], scale=scale)
    got, got_lse = kv_attention(q.to(DEV), device_cache4(parts), table.to(DEV), torch.tensor([L], dtype=torch.int32, device=DEV),
                                offsets([many]).to(DEV), scale=scale, return_lse=True)
    largest = 6 * 2.0 ** max(top, rest)
    bound = tol + L * largest * 2.0 ** (-39 if many < 20 else -37)
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    assert ((got_lse.cpu().double() - lse).abs() <= tol_lse).all()
    if rest == 0 and math.exp(-nats) * L < 2.0 ** -6:        # nothing of this shows at a spread of 2^14
        assert (off <= tol + 2.0 ** -22).all()
