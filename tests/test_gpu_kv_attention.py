"""kv_attention against 64-bit attention over the cache's values, element by element, within the bounds
that 32-bit scores and 11-bit weights give (serving.attention)."""
import math

import pytest
import torch

from polar_pack_amd.kv_cache import kv_attention
from serving import DEV, attention, device_cache, offsets, random_cache, tables

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16


def check(H, G, D, bs, codes, value, lens, news, *, causal=True, window=0, scale=None, width=None, edit=None, cu=True,
          q_scale=1.0, extra=0):
    g = torch.Generator().manual_seed(H * 1000 + D + bs + sum(lens) + sum(news))
    pages = sum(-(-max(n, 0) // bs) for n in lens) + 2
    parts = random_cache(pages, H, bs, D, codes, g)
    table = tables(lens, bs, pages, g, width)
    q = (torch.randn(sum(news) + extra, H * G, D, generator=g) * q_scale).to(value)
    if edit:
        edit(parts, table, q)
    want, lse, tol, tol_lse = attention(q, parts, table, lens, news, causal, window, scale)
    got, got_lse = kv_attention(q.to(DEV), device_cache(parts), table.to(DEV),
                                torch.tensor(lens, dtype=torch.int32, device=DEV),
                                offsets(news).to(DEV) if cu else None, causal=causal, window=window, scale=scale,
                                return_lse=True)
    got, got_lse = got.cpu().double(), got_lse.cpu().double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan())
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol.clamp(min=1e-30)).nan_to_num(0).max()),
                           bad.nonzero()[:3].tolist())
    both = (got_lse == lse) | (got_lse.isnan() & lse.isnan()) | ((got_lse - lse).abs() <= tol_lse)
    assert both.all(), (got_lse - lse).abs().max()
    return got


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("H,G,D,bs", [(2, 8, 128, 64), (1, 1, 64, 16), (3, 4, 64, 32), (1, 16, 256, 128), (2, 3, 192, 64),
                                      (1, 5, 128, 16), (1, 24, 128, 32)])
def test_single_tokens(H, G, D, bs, codes, value):
    lens = [1, 2, 15, 16, 63, 64, 65, 200, 333]
    check(H, G, D, bs, codes, value, lens, [1] * len(lens), cu=False)


@pytest.mark.parametrize("G,D", [(33, 64), (40, 128), (128, 64), (130, 128)])
def test_single_tokens_of_wide_groups(G, D):
    """More query heads a key head than the few-row kernel takes."""
    check(1, G, D, 64, INT8, F16, [1, 64, 65, 200, 777], [1] * 5, cu=False)


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("G,new,window", [(4, 2, 0), (8, 4, 50), (4, 28, 0), (4, 80, 70)])
def test_every_kernel(G, new, window, D, bs, value, codes):
    """Every compiled form of the two kernels, at 8, 32, 112 and 320 rows a sequence and head: ragged lengths, the longest of
    several runs, one sequence without tokens and one as long as its tokens."""
    lens, news = [new + 231, 7, new, new + 65], [new, 0, new, max(1, new - 3)]
    check(2, G, D, bs, codes, value, lens, news, window=window, extra=1)


@pytest.mark.parametrize("codes,value", [(INT8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("L", [1023, 1024, 4097, 20000])
def test_one_long_sequence(L, codes, value):
    check(1, 8, 128, 64, codes, value, [L], [1], cu=False)


@pytest.mark.parametrize("codes,value", [(INT8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("H,G,D,bs", [(2, 8, 128, 64), (1, 1, 64, 16), (2, 4, 64, 128), (1, 2, 256, 32), (1, 3, 192, 16)])
def test_few_tokens(H, G, D, bs, codes, value):
    lens, news = [5, 70, 257, 3, 600], [5, 2, 7, 1, 3]
    check(H, G, D, bs, codes, value, lens, news)


@pytest.mark.parametrize("codes,value", [(INT8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("H,G,D,bs", [(2, 8, 128, 64), (1, 1, 64, 16), (1, 4, 64, 32), (1, 2, 256, 64), (1, 3, 192, 128)])
def test_prompts(H, G, D, bs, codes, value):
    """Whole prompts, prompts behind a cached prefix, ragged, with single tokens among them."""
    lens, news = [300, 517, 1, 130, 64], [300, 200, 1, 129, 64]
    check(H, G, D, bs, codes, value, lens, news)


@pytest.mark.parametrize("codes,value", [(INT8, F16), (INT8, BF16), (E4M3, F16), (E4M3, BF16)])
@pytest.mark.parametrize("D", [192, 256])
@pytest.mark.parametrize("bs", [16, 32])
def test_prompts_of_wide_heads_in_small_pages(bs, D, codes, value):
    """Where the many-row kernel has the fewest registers to spare; several row tiles a workgroup."""
    check(2, 2, D, bs, codes, value, [450, 150, 40], [150, 150, 30])
    check(1, 2, D, bs, codes, value, [450, 150, 40], [150, 150, 30], causal=False)


@pytest.mark.parametrize("G", [1, 8])
def test_prompt_piece_behind_a_long_prefix(G):
    check(1, G, 128, 64, INT8, F16, [5003], [150])


@pytest.mark.parametrize("news", [[1, 1, 1], [4, 40, 3], [150, 200, 90]])
@pytest.mark.parametrize("window", [1, 16, 100, 10 ** 6])
def test_window(window, news):
    check(2, 4, 64, 16, INT8, F16, [300, 201, 90], news, window=window)


@pytest.mark.parametrize("news", [[1, 1, 1], [4, 40, 3], [150, 200, 90]])
def test_every_key(news):
    check(2, 4, 128, 32, E4M3, F16, [300, 201, 90], news, causal=False)


@pytest.mark.parametrize("G,piece", [(4, 40), (1, 20), (4, 3)])
def test_queries_of_another_text(G, piece):
    """150 queries to 40 keys: in calls of at most 40 each sees them all; in one call only the last 40 have a
    position, and the others see nothing."""
    g = torch.Generator().manual_seed(piece)
    parts = random_cache(3, 1, 16, 64, INT8, g)
    table = tables([40], 16, 3, g)
    q = torch.randn(150, G, 64, generator=g).half()
    cache, at = device_cache(parts), (table.to(DEV), torch.tensor([40], dtype=torch.int32, device=DEV))
    want, tol = (torch.cat(x) for x in zip(*[attention(q[i:i + 40], parts, table, [40], [len(q[i:i + 40])], False)[::2]
                                             for i in range(0, 150, 40)]))
    got = torch.cat([kv_attention(x.to(DEV), cache, *at, offsets([len(x)]).to(DEV), causal=False)
                     for x in q.split(piece)]).cpu().double()
    assert ((got - want).abs() <= tol).all()
    whole, lse = kv_attention(q.to(DEV), cache, *at, offsets([150]).to(DEV), causal=False, return_lse=True)
    assert ((whole[110:].cpu().double() - want[110:]).abs() <= tol[110:]).all()
    assert not whole[:110].any() and (lse[:110] == -math.inf).all() and lse[110:].isfinite().all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("many", [1, 30])
def test_rows_that_see_nothing(causal, many):
    """Empty sequences, lengths below the number of tokens, pages out of range, tokens past the table,
    tokens past the last sequence."""
    def edit(parts, table, q):
        table[2, 0] = -1                   # a whole sequence's page
        table[4, 1] = 10 ** 6
    lens, news = [0, 3, 10, 400, 160], [many, 4 + many, many, 3, many]
    got = check(2, 4, 64, 64, INT8, F16, lens, news, causal=causal, edit=edit, width=4, extra=5)
    assert not got[:many].any() and not got[-5:].any()


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("many", [1, 20, 150])
def test_what_lies_behind_a_mask_does_not_matter(codes, many):
    """Codes that are NaN (e4m3) and scales that are infinite or NaN past the length, or in pages that a
    window hides, reach no row; a page that is seen makes its rows NaN."""
    bs = 16
    def edit(parts, table, q):
        k, v, ks, vs = parts
        p = int(table[0, -1])
        k.view(torch.int8)[p, :, 5:] = 127                     # e4m3: NaN, past the length
        v.view(torch.int8)[p, :, :, 5:] = 127
        for t in (ks, vs):
            t[int(table[0, 0])] = math.nan                     # outside the window
            t[int(table[0, 1])] = math.inf
    L = 16 * bs + 5 + (16 * bs if many > 20 else 0)
    got = check(1, 4, 64, bs, codes, F16, [L], [many], window=20, edit=edit)
    assert not got.isnan().any()

    def edit2(parts, table, q):
        parts[3][int(table[0, 3])] = math.nan
    got = check(1, 4, 64, bs, codes, F16, [L], [many], edit=edit2)
    assert got.isnan().all()


@pytest.mark.parametrize("many", [1, 150])
def test_scales_far_apart(many):
    """Values and keys of pages thousands of times larger or smaller than their neighbours'."""
    def edit(parts, table, q):
        g = torch.Generator().manual_seed(4)
        parts[3][:] = 10.0 ** torch.randint(-6, 4, parts[3].shape, generator=g).float()
        parts[2][:] *= 10.0 ** torch.randint(-4, 1, parts[2].shape, generator=g).float()
    check(1, 8, 128, 64, INT8, BF16, [900], [many], edit=edit)


@pytest.mark.parametrize("many", [1, 150])
@pytest.mark.parametrize("large", [0, 1])
def test_value_scales_as_far_apart_as_they_may_be(large, many):
    """The pages of the smaller scale add nothing to the values but count in the sum of weights."""
    def edit(parts, table, q):
        of = table[0].long()
        parts[3][of[large::2]] = 2.0 ** 40
        parts[3][of[1 - large::2]] = 2.0 ** -60
    check(1, 8, 128, 64, INT8, BF16, [900], [many], edit=edit)


@pytest.mark.parametrize("many", [1, 150])
@pytest.mark.parametrize("value,q_scale", [(F16, 1e-6), (F16, 2000.0), (BF16, 1e-30), (BF16, 1e6)])
def test_queries_of_any_size(value, q_scale, many):
    """Subnormal and huge queries; with huge ones a row is one key's value."""
    check(1, 8, 128, 64, INT8, value, [300], [many], q_scale=q_scale, scale=1.0 / (q_scale * 10))
    check(1, 8, 128, 64, INT8, value, [300], [many], q_scale=q_scale, scale=0.0)


@pytest.mark.parametrize("many", [1, 150])
@pytest.mark.parametrize("value,small", [(BF16, -12), (BF16, -30), (F16, -9)])
def test_queries_of_unequal_channels(value, small, many):
    """Channels of 2^small to 2^(small + 1) beside one of 1, whose keys are zero: the scores are the small ones', and
    to 2^-30 of the largest they keep all their bits."""
    def edit(parts, table, q):
        parts[0][..., 0] = 0
        q.copy_(torch.copysign(q.abs() % 1 + 1, q) * 2.0 ** small)
        q[..., 0] = 1
    check(1, 8, 128, 64, INT8, value, [300], [many], edit=edit, scale=2.0 ** -small / 8)


def one_score(codes, size, keys, many, marked=None):
    """Attention of ``many`` tokens, the last of ``keys``, to keys that all have the score ``size`` (base 2), except
    that with ``marked`` all but that one have -``size``; and the values."""
    g = torch.Generator().manual_seed(keys + many)
    parts = random_cache(-(-keys // 64), 1, 64, 64, codes, g)
    parts[0].copy_((torch.full(parts[0].shape, 100.0 if marked is None else -100.0)).to(codes))
    if marked is not None:
        parts[0][marked // 64, 0, marked % 64] = torch.full((64,), 100.0).to(codes)
    for t in parts[2:]:
        t.fill_(2.0 ** -6)
    table = torch.arange(-(-keys // 64), dtype=torch.int32)[None]
    q = torch.ones(many, 4, 64, dtype=torch.float16)
    code = float(parts[0].double().abs().max())
    got, lse = kv_attention(q.to(DEV), device_cache(parts), table.to(DEV),
                            torch.tensor([keys], dtype=torch.int32, device=DEV), offsets([many]).to(DEV),
                            scale=size * math.log(2) / (code * 64 * 2.0 ** -6), return_lse=True)
    values = parts[1][:, 0].double().transpose(1, 2).reshape(-1, 64) * 2.0 ** -6
    return got.cpu().double(), lse.cpu().double(), values


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("many", [1, 12, 150])
@pytest.mark.parametrize("size", [2.0 ** e * f for e in (23, 24, 25, 26, 27, 28, 40) for f in (1.01, 1.3, 1.9)])
def test_scores_that_are_large(size, many, codes):
    """Where neighbouring floats are 1 to 16 apart, and beyond: weights are still at most what fp16 holds, and the
    key that is ahead has all of it."""
    got, lse, values = one_score(codes, size, 300, many, marked=70)
    assert ((got - values[70]).abs() <= 2.0 ** -11 * values[70].abs()).all()
    assert ((lse - size * math.log(2)).abs() <= 2.0 ** -20 * size).all()


@pytest.mark.parametrize("many", [1, 12, 60])
@pytest.mark.parametrize("size", [-1e29, -1e31, -3e37, 1e31])
def test_scores_as_large_as_floats(size, many):
    """A row whose scores are all far below zero sees its keys all the same."""
    got, lse, values = one_score(INT8, size, 64, many)
    for i in range(many):
        seen = values[:64 - many + 1 + i]
        want, mass = seen.mean(0), seen.abs().mean(0)
        assert ((got[i] - want).abs() <= 2.0 ** -11 * (want.abs() + mass) + 2.0 ** -20 * mass).all()
    assert ((lse - size * math.log(2)).abs() <= 2.0 ** -20 * abs(size)).all()


@pytest.mark.parametrize("many", [1, 150])
def test_queries_that_are_not_finite(many):
    def edit(parts, table, q):
        q[0, 0, 3] = math.nan
        q[0, 1, 3] = math.inf
    g = torch.Generator().manual_seed(1)
    parts = random_cache(8, 1, 64, 64, INT8, g)
    table = tables([300], 64, 8, g)
    q = torch.randn(many, 4, 64, generator=g).half()
    clean = q.clone()
    edit(parts, table, q)
    args = (device_cache(parts), table.to(DEV), torch.tensor([300], dtype=torch.int32, device=DEV),
            offsets([many]).to(DEV))
    a, b = kv_attention(q.to(DEV), *args), kv_attention(clean.to(DEV), *args)
    assert a[0, :2].isnan().all()
    assert torch.equal(a[0, 2:], b[0, 2:]) and torch.equal(a[1:], b[1:])


def test_strides_of_queries():
    g = torch.Generator().manual_seed(9)
    parts = random_cache(12, 2, 64, 128, INT8, g)
    for news in ([1, 1], [100, 30]):
        lens = [300, 200]
        table = tables(lens, 64, 12, g).to(DEV)
        cache, n = device_cache(parts), sum(news)
        L, cu = torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV)
        q = torch.randn(n, 8, 128, generator=g).half().to(DEV)
        want = kv_attention(q, cache, table, L, cu)
        for pad, off in ((4, 1), (16, 8)):
            wide = torch.zeros(n, 8 * 128 + pad, dtype=torch.float16, device=DEV)
            part = wide[:, off:off + 1024].view(n, 8, 128)
            part.copy_(q)
            assert torch.equal(kv_attention(part, cache, table, L, cu), want)
        by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(kv_attention(by_head, cache, table, L, cu), want)
        wide_table = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
        wide_table[:, :table.shape[1]] = table
        again = kv_attention(q, cache, wide_table[:, :30], L, cu)
        assert (again.float() - want.float()).abs().max() <= 2.0 ** -9 * want.float().abs().max()


def test_queries_that_negate_when_they_are_read():
    g = torch.Generator().manual_seed(15)
    parts = random_cache(12, 2, 64, 64, INT8, g)
    cache = device_cache(parts)
    for news in ([1, 1], [100, 30]):
        table, L = tables([300, 200], 64, 12, g).to(DEV), torch.tensor([300, 200], dtype=torch.int32, device=DEV)
        q = torch.randn(sum(news), 8, 64, generator=g).half().to(DEV)
        view = torch._neg_view(-q)
        assert view.is_neg() and torch.equal(view, q)
        args = (cache, table, L, offsets(news).to(DEV))
        assert torch.equal(kv_attention(view, *args), kv_attention(q, *args))


def test_shared_pages():
    """Two sequences with one prefix: the same rows."""
    g = torch.Generator().manual_seed(6)
    parts = random_cache(6, 2, 64, 128, E4M3, g)
    table = torch.tensor([[0, 1, 2], [0, 1, 2], [0, 1, 4]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 8, 128, generator=g).half().expand(3, 8, 128).to(DEV)
    out = kv_attention(q, device_cache(parts), table, torch.tensor([150, 150, 120], dtype=torch.int32, device=DEV))
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])


def test_many_sequences():
    g = torch.Generator().manual_seed(8)
    news = torch.randint(0, 4, (150,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 50, (150,), generator=g))]
    check(1, 4, 64, 16, INT8, F16, lens, news)


def test_more_sequences_than_are_dealt():
    """Past 1,020 sequences every row tile is one workgroup's."""
    g = torch.Generator().manual_seed(12)
    lens = torch.randint(0, 90, (1100,), generator=g).tolist()
    check(1, 4, 64, 64, INT8, F16, lens, [1] * 1100, cu=False)
    check(1, 4, 64, 64, E4M3, F16, lens, [min(n, 2) for n in lens])


@pytest.mark.parametrize("B,n", [(70, 68), (20, 240)])
def test_many_row_tiles(B, n):
    """Row tiles enough for every CU are not shared; those that see the most keys come first."""
    g = torch.Generator().manual_seed(B)
    news = torch.randint(n - 20, n + 20, (B,), generator=g).tolist()
    news[3], news[5] = 1, 0
    assert sum(news) * 32 / 256 >= 2 * torch.cuda.get_device_properties(DEV).multi_processor_count
    check(1, 32, 64, 64, INT8, BF16, [m + 30 * (i % 3) for i, m in enumerate(news)], news, extra=3)


@pytest.mark.parametrize("codes,value", [(INT8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("H,G,D,bs,kw", [(1, 2, 192, 64, {}), (2, 4, 256, 64, {}), (1, 2, 256, 16, {"window": 90}),
                                         (1, 4, 192, 32, {"causal": False}), (2, 2, 128, 128, {}),
                                         (1, 3, 64, 16, {"window": 70})])
def test_row_tiles_of_four_wavefronts(H, G, D, bs, kw, codes, value):
    """At 65-128 rows a sequence and head, and at 192 and 256 values a head for more too, a workgroup is 4
    wavefronts and its ring of keys has two slots: each wavefront has read the first tile of keys before any
    writes the third over it.  Prompts of one to eight tiles, several row tiles a workgroup."""
    n = 50 if D <= 128 else 150
    lens, news = [n + 300, n, n + 30, 3 * n + 64, n + 1], [n, n, n - 3, n + 5, 1]
    check(H, G, D, bs, codes, value, lens, news, **kw)


@pytest.mark.parametrize("codes,value,D,window", [(INT8, F16, 256, 0), (E4M3, BF16, 192, 40), (E4M3, F16, 128, 0)])
def test_many_row_tiles_of_four_wavefronts(codes, value, D, window):
    """The same with row tiles enough for every CU, which are not shared; 96-124 rows a sequence and head at 128
    values a head."""
    B, n, G = (170, 3, 32) if D == 128 else (21, 25, 32)
    H = 4
    g = torch.Generator().manual_seed(D)
    news = torch.randint(n, n + 2, (B,), generator=g).tolist()
    while sum(news) * H * G / 128 < 2 * torch.cuda.get_device_properties(DEV).multi_processor_count:
        news = [x + 1 for x in news]
    check(H, G, D, 64, codes, value, [m + 60 * (i % 3) for i, m in enumerate(news)], news, window=window, extra=2)


@pytest.mark.parametrize("G,D,news", [(4, 64, [20, 25]), (4, 256, [150, 90]), (8, 128, [150, 90])])
def test_one_answer_of_many_rows(G, D, news):
    g = torch.Generator().manual_seed(D)
    parts = random_cache(110, 2, 64, D, INT8, g)
    lens = [5000, 777]
    table = tables(lens, 64, 110, g).to(DEV)
    cache, L, cu = device_cache(parts), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV)
    q = torch.randn(sum(news), 2 * G, D, generator=g).half().to(DEV)
    want = kv_attention(q, cache, table, L, cu)
    for _ in range(5):
        assert torch.equal(kv_attention(q, cache, table, L, cu), want)


def test_one_answer():
    """Joins do not depend on the order in which parts of a row end."""
    g = torch.Generator().manual_seed(3)
    parts = random_cache(600, 2, 64, 128, INT8, g)
    lens = [20000, 777]
    table = tables(lens, 64, 600, g).to(DEV)
    cache, L = device_cache(parts), torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(2, 16, 128, generator=g).half().to(DEV)
    want = kv_attention(q, cache, table, L)
    for _ in range(5):
        assert torch.equal(kv_attention(q, cache, table, L), want)


@pytest.mark.parametrize("news", [[1, 1], [90, 60]])
def test_in_a_graph_and_on_another_stream(news):
    g = torch.Generator().manual_seed(31)
    parts = random_cache(80, 2, 64, 128, INT8, g)
    lens = [3000, 900]
    table = tables(lens, 64, 80, g).to(DEV)
    cache, L = device_cache(parts), torch.tensor(lens, dtype=torch.int32, device=DEV)
    cu = None if sum(news) == 2 else offsets(news).to(DEV)
    q = torch.randn(sum(news), 16, 128, generator=g).half().to(DEV)
    want = kv_attention(q, cache, table, L, cu)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = kv_attention(q, cache, table, L, cu)
    side.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_attention(q, cache, table, L, cu)
    first = q.clone()
    for i in range(4):
        q.copy_(first * (1 + i))
        L.copy_(torch.tensor([3000 - 64 * i, 900], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kv_attention(q, cache, table, L, cu)), i


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB of codes, its pages at both ends."""
    H, D, bs, pages = 8, 128, 128, 36000
    from polar_pack_amd.kv_cache import KVCache, kv_append
    cache = KVCache.zeros(pages, H, D, block=bs, device=DEV)
    assert cache.k.numel() > 2 ** 32
    table = torch.tensor([[pages - 1, 0, pages - 2, 1]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(1)
    n = 400
    k, v, q = (torch.randn(n, H, D, generator=g).half() for _ in range(3))
    L, cu = torch.tensor([n], dtype=torch.int32, device=DEV), offsets([n]).to(DEV)
    kv_append(cache, k.to(DEV), v.to(DEV), table, L, cu)
    used = table[0].long()
    parts = [t.view(torch.int8)[used].cpu().view(t.dtype) if t.dtype != torch.float32 else t[used].cpu()
             for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    own = torch.arange(4, dtype=torch.int32)[None]
    for rows in (n, 1):
        want, _, tol, _ = attention(q[-rows:], parts, own, [n], [rows])
        got = kv_attention(q[-rows:].to(DEV), cache, table, L, offsets([rows]).to(DEV)).cpu().double()
        assert ((got - want).abs() <= tol).all()


def test_refusals():
    g = torch.Generator().manual_seed(0)
    cache = device_cache(random_cache(2, 2, 16, 64, INT8, g))
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(TypeError):
        kv_attention(q.float(), cache, table, lens)
    with pytest.raises(ValueError):
        kv_attention(q[:, :3], cache, table, lens)
    with pytest.raises(ValueError):
        kv_attention(q[..., :32], cache, table, lens)
    with pytest.raises(ValueError):
        kv_attention(q, cache, table, lens, window=-1)
    with pytest.raises(ValueError):
        kv_attention(q, cache, table, lens, window=5, causal=False)
    with pytest.raises(ValueError):
        kv_attention(q[:1], cache, table, lens)
    with pytest.raises(ValueError):
        kv_attention(q.cpu(), cache, table, lens)
    none = kv_attention(q[:0], cache, table, lens, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert none.shape == (0, 4, 64)
