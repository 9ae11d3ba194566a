"""kv_attention over the 4-bit cache against 64-bit attention over the values its codes stand for, within the bounds that
32-bit scores and 11-bit weights give (serving.attention); codes times scales are exact in the kernels."""
import math

import pytest
import torch

from polar_pack_amd.kv_cache import kv_append, kv_attention, kv_read, kv_rotate_append
from polar_pack_amd.rotary import Rotary
from serving import DEV, attention, offsets, tables
from serving4 import device_cache4, f8, plain_parts, random_cache4, value4

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def check(H, G, D, bs, value, lens, news, *, causal=True, window=0, scale=None, width=None, edit=None, cu=True, q_scale=1.0,
          extra=0, low=-3, high=1):
    g = torch.Generator().manual_seed(H * 1000 + D + bs + sum(lens) + sum(news))
    pages = sum(-(-max(n, 0) // bs) for n in lens) + 2
    parts = random_cache4(pages, H, bs, D, g, low, high)
    table = tables(lens, bs, pages, g, width)
    q = (torch.randn(sum(news) + extra, H * G, D, generator=g) * q_scale).to(value)
    if edit:
        edit(parts, table, q)
    want, lse, tol, tol_lse = attention(q, plain_parts(parts), table, lens, news, causal, window, scale)
    got, got_lse = kv_attention(q.to(DEV), device_cache4(parts), table.to(DEV),
                                torch.tensor(lens, dtype=torch.int32, device=DEV),
                                offsets(news).to(DEV) if cu else None, causal=causal, window=window, scale=scale,
                                return_lse=True)
    got, got_lse = got.cpu().double(), got_lse.cpu().double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan())
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol.clamp(min=1e-30)).nan_to_num(0).max()),
                           bad.nonzero()[:3].tolist())
    both = (got_lse == lse) | (got_lse.isnan() & got.isnan().any(-1)) | ((got_lse - lse).abs() <= tol_lse)
    assert both.all(), (got_lse - lse).abs().max()
    return got


@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("H,G,D,bs", [(2, 8, 128, 64), (1, 1, 64, 16), (3, 4, 64, 32), (1, 16, 256, 128), (2, 3, 192, 64),
                                      (1, 5, 128, 16), (1, 24, 128, 32)])
def test_single_tokens(H, G, D, bs, value):
    lens = [1, 2, 15, 16, 63, 64, 65, 200, 333]
    check(H, G, D, bs, value, lens, [1] * len(lens), cu=False)


@pytest.mark.parametrize("G,D", [(33, 64), (40, 128), (128, 64), (130, 128)])
def test_single_tokens_of_wide_groups(G, D):
    check(1, G, D, 64, F16, [1, 64, 65, 200, 777], [1] * 5, cu=False)


@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("G,new,window", [(4, 2, 0), (8, 4, 50), (4, 28, 0), (4, 80, 70)])
def test_every_kernel(G, new, window, D, bs, value):
    """Every compiled form of the two kernels, at 8, 32, 112 and 320 rows a sequence and head: ragged lengths, the longest of
    several runs, one sequence without tokens and one as long as its tokens."""
    lens, news = [new + 231, 7, new, new + 65], [new, 0, new, max(1, new - 3)]
    check(2, G, D, bs, value, lens, news, window=window, extra=1)


@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("L", [1023, 1024, 4097, 20000])
def test_one_long_sequence(L, value):
    check(1, 8, 128, 64, value, [L], [1], cu=False)


@pytest.mark.parametrize("H,G,D,bs", [(2, 8, 128, 64), (1, 1, 64, 16), (2, 4, 64, 128), (1, 2, 256, 32), (1, 3, 192, 16)])
def test_few_tokens(H, G, D, bs):
    check(H, G, D, bs, BF16, [5, 70, 257, 3, 600], [5, 2, 7, 1, 3])


@pytest.mark.parametrize("H,G,D,bs", [(2, 8, 128, 64), (1, 1, 64, 16), (1, 4, 64, 32), (1, 2, 256, 64), (1, 3, 192, 128)])
def test_prompts(H, G, D, bs):
    """Whole prompts, prompts behind a cached prefix, ragged, with single tokens among them."""
    check(H, G, D, bs, F16, [300, 517, 1, 130, 64], [300, 200, 1, 129, 64])


@pytest.mark.parametrize("D", [192, 256])
@pytest.mark.parametrize("bs", [16, 32])
def test_prompts_of_wide_heads_in_small_pages(bs, D):
    check(2, 2, D, bs, F16, [450, 150, 40], [150, 150, 30])
    check(1, 2, D, bs, BF16, [450, 150, 40], [150, 150, 30], causal=False)


@pytest.mark.parametrize("news", [[1, 1, 1], [4, 40, 3], [150, 200, 90]])
@pytest.mark.parametrize("window", [1, 16, 100, 10 ** 6])
def test_window(window, news):
    check(2, 4, 64, 16, F16, [300, 201, 90], news, window=window)


@pytest.mark.parametrize("news", [[1, 1, 1], [4, 40, 3], [150, 200, 90]])
def test_every_key(news):
    check(2, 4, 128, 32, F16, [300, 201, 90], news, causal=False)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("many", [1, 30])
def test_rows_that_see_nothing(causal, many):
    def edit(parts, table, q):
        table[2, 0] = -1                   # a whole sequence's page
        table[4, 1] = 10 ** 6
    lens, news = [0, 3, 10, 400, 160], [many, 4 + many, many, 3, many]
    got = check(2, 4, 64, 64, F16, lens, news, causal=causal, edit=edit, width=4, extra=5)
    assert not got[:many].any() and not got[-5:].any()


@pytest.mark.parametrize("what", [0x7f, 0x7c, 0xff, 0x7b])
@pytest.mark.parametrize("many", [1, 20, 150])
def test_what_lies_behind_a_mask_does_not_matter(many, what):
    """Scales that are NaN, infinite or huge past the length, or of keys that a window hides, reach no row."""
    bs = 16

    def edit(parts, table, q):
        k, v, ks, vs = parts
        last, first = int(table[0, -1]), int(table[0, 0])
        ks.view(torch.uint8)[last, :, 5:] = what
        vs.view(torch.uint8)[last, :, :, 5:] = what
        ks.view(torch.uint8)[first, :, 3:9] = what
    L = 16 * bs + 5 + (16 * bs if many > 20 else 0)
    got = check(1, 4, 64, bs, F16, [L], [many], window=20, edit=edit)
    assert not got.isnan().any()


@pytest.mark.parametrize("many", [1, 30, 150])
def test_a_token_that_is_not_finite(many):
    """Rows that see it are NaN, rows before it and of the other head are not."""
    at = 400 - many // 2 - 1

    def edit(parts, table, q):
        parts[2].view(torch.uint8)[int(table[0, at // 16]), 1, at % 16] = 0x7f
    got = check(2, 4, 64, 16, F16, [400], [many], edit=edit)
    sees = torch.arange(400 - many, 400) >= at
    assert torch.equal(got[:, 4:].isnan().all(-1), sees[:, None].expand(many, 4))
    assert not got[:, :4].isnan().any() and not got[~sees].isnan().any()


@pytest.mark.parametrize("many", [1, 150])
@pytest.mark.parametrize("low,high", [(-14, -13), (13, 14), (-14, 14), (-14, -8)])
def test_scales_of_any_size(low, high, many):
    """The whole range, all in one cache and alone; scores held to a few units by the scale of the scores."""
    check(1, 8, 128, 64, BF16, [500], [many], low=low, high=high, scale=2.0 ** -high / 40)


@pytest.mark.parametrize("many", [1, 150])
@pytest.mark.parametrize("value,q_scale", [(F16, 1e-6), (F16, 2000.0), (BF16, 1e-30), (BF16, 1e6)])
def test_queries_of_any_size(value, q_scale, many):
    check(1, 8, 128, 64, value, [300], [many], q_scale=q_scale, scale=1.0 / (q_scale * 10))
    check(1, 8, 128, 64, value, [300], [many], q_scale=q_scale, scale=0.0)


@pytest.mark.parametrize("many", [1, 12, 150])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 25 * 1.3, 2.0 ** 40 * 1.9])
def test_scores_that_are_large(size, many):
    """One key far ahead of the others: its value is the answer."""
    g = torch.Generator().manual_seed(many)
    parts = random_cache4(5, 1, 64, 64, g, 0, 1)
    parts[0].fill_(0xaa)                                     # -1 everywhere, and 1 at one key
    parts[0][1, 0, 6] = 0x22
    table = torch.arange(5, dtype=torch.int32)[None]
    q = torch.ones(many, 4, 64, dtype=F16)
    got, lse = kv_attention(q.to(DEV), device_cache4(parts), table.to(DEV), torch.tensor([300], dtype=torch.int32, device=DEV),
                            offsets([many]).to(DEV), scale=size * math.log(2) / 64, return_lse=True)
    want = plain_parts(parts)[1][1, 0, :, 6]
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -11 * want.abs()).all()
    assert ((lse.cpu().double() - size * math.log(2)).abs() <= 2.0 ** -20 * size).all()


def test_pages_at_the_end_of_a_large_cache():
    """Offsets past 2^32 bytes of codes: the last pages of a cache of 9 GB."""
    H, D, bs, pages = 8, 128, 64, 2 ** 17
    from polar_pack_amd.kv_cache import KVCache4
    g = torch.Generator().manual_seed(3)
    parts = random_cache4(4, H, bs, D, g)
    k = torch.empty(pages, H, bs, D // 2, dtype=torch.uint8, device=DEV)
    v = torch.empty(pages, H, D, bs // 2, dtype=torch.uint8, device=DEV)
    ks = torch.empty(pages, H, bs, D // 32, dtype=torch.uint8, device=DEV)
    vs = torch.empty(pages, H, D // 32, bs, dtype=torch.uint8, device=DEV)
    for t, p in zip((k, v, ks, vs), parts):
        t[-4:] = p.view(torch.uint8).to(DEV)
    cache = KVCache4(k, v, ks.view(torch.float8_e5m2), vs.view(torch.float8_e5m2))
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32)
    for news in ([1], [150]):
        q = torch.randn(news[0], H * 2, D, generator=g).half()
        want, _, tol, _ = attention(q, plain_parts(parts), table, [250], news)
        got = kv_attention(q.to(DEV), cache, (table + pages - 4).to(DEV), torch.tensor([250], dtype=torch.int32, device=DEV),
                           offsets(news).to(DEV))
        assert ((got.cpu().double() - want).abs() <= tol).all()
    new = torch.randn(2, 3, H, D, generator=g).half().to(DEV)
    at = ((table + pages - 4).to(DEV), torch.tensor([203], dtype=torch.int32, device=DEV), offsets([3]).to(DEV))
    small = device_cache4(parts)
    kv_append(cache, *new, *at)
    kv_append(small, *new, table.to(DEV), *at[1:])
    assert torch.equal(cache.k[-4:], small.k) and torch.equal(cache.v[-4:], small.v)
    for a, b in zip(kv_read(cache, *at, total=3), kv_read(small, table.to(DEV), *at[1:], total=3)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("news", [[1, 1], [5, 3], [200, 40]])
def test_a_step_as_a_model_runs_it(news):
    """Turn, append, attend, twice with the same answers; against plain attention over what the cache then holds; in a
    graph that is replayed with eager calls between."""
    H, D, bs, lens = 2, 128, 16, [230, 90]
    g = torch.Generator().manual_seed(sum(news))
    parts = random_cache4(24, H, bs, D, g)
    table = tables(lens, bs, 24, g)
    n = sum(news)
    q, k, v = (torch.randn(n, h, D, generator=g).half().to(DEV) for h in (8 * H, H, H))
    t, ln, cu, r = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV), Rotary(D)
    cache = device_cache4(parts)

    def step(c):
        turned = kv_rotate_append(c, q, k, v, r, t, ln, cu)
        return turned, kv_attention(turned, c, t, ln, cu)
    turned, out = step(cache)
    now = [x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    want, _, tol, _ = attention(turned.cpu(), plain_parts(now), table, lens, news)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert torch.equal(step(cache)[1], out)
    graph, other = torch.cuda.CUDAGraph(), device_cache4(parts)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _, replayed = step(other)
    for i in range(4):
        for x in (q, k, v):
            x.normal_()
        want = step(cache)[1]
        replayed.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed, want), i
