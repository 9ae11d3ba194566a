"""kv_append and kv_read: codes and scales against the float32 definition bit for bit (every step of it
is a correctly rounded operation), values against the appended ones in 64 bits."""
import math

import pytest
import torch

from polar_pack_amd.kv_cache import KVCache, kv_append, kv_read
from serving import DEV, append, device_cache, gather, offsets, random_cache, raw, tables

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]


def same(cache, want, ctx=""):
    for name, w in zip(("k", "v", "k_scale", "v_scale"), want):
        got = getattr(cache, name).cpu()
        if got.dtype != torch.float32:
            got, w = raw(got), raw(w)
        assert torch.equal(got.nan_to_num(7.0) if got.dtype == torch.float32 else got,
                           w.nan_to_num(7.0) if w.dtype == torch.float32 else w), f"{ctx} {name}"


def problem(H, D, bs, dtype, lens, news, seed, value=torch.float16, grow=1.0):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(n, 0) // bs) for n in lens) + 2
    parts = random_cache(pages, H, bs, D, dtype, g)
    table = tables(lens, bs, pages, g)
    n = sum(news)
    k, v = (torch.randn(n, H, D, generator=g).mul_(grow).to(value) for _ in range(2))
    return parts, table, k, v


def call(parts, table, k, v, lens, news, cu=True):
    cache = device_cache(parts)
    kv_append(cache, k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
              offsets(news).to(DEV) if cu else None)
    return cache


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("value", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,D,bs", [(2, 128, 64), (1, 64, 16), (3, 256, 128), (2, 192, 32), (1, 192, 16)])
def test_append_matches_the_definition(H, D, bs, dtype, value):
    lens, news = [1, bs, bs + 1, 3 * bs - 1, 2 * bs + 5], [1, bs, 2, 2 * bs + 3, 5]
    parts, table, k, v = problem(H, D, bs, dtype, lens, news, D + bs, value)
    same(call(parts, table, k, v, lens, news), append(parts, k, v, table, lens, news))


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("value", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_every_kernel(D, bs, value, dtype):
    """Every compiled form of append and read: a new page, the end of a page and the next, a whole page and a piece."""
    lens, news = [3, bs + 2, 2 * bs, bs - 1], [3, 5, bs, 2]
    parts, table, k, v = problem(2, D, bs, dtype, lens, news, D + bs, value)
    want = append(parts, k, v, table, lens, news)
    cache = call(parts, table, k, v, lens, news)
    same(cache, want)
    for out in (torch.float16, torch.bfloat16, torch.float32):
        got = kv_read(cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV),
                      total=sum(news), dtype=out)
        at = 0
        for b, n in enumerate(news):
            for h in range(2):
                for x, full in zip(got, gather(want, table[b], lens[b], h)[:2]):
                    assert torch.equal(x[at:at + n, h].cpu(), full[lens[b] - n:].float().to(out)), (b, h, out)
            at += n


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("grow", [1e-3, 1.0, 300.0])
def test_single_tokens_where_the_scale_grows_or_not(dtype, grow):
    """One token a sequence at every kind of place in a page: the first, in the middle, the last."""
    H, D, bs = 2, 128, 64
    lens, news = [1, 2, 37, 64, 65, 128, 100], [1] * 7
    parts, table, k, v = problem(H, D, bs, dtype, lens, news, 3, torch.float16, grow)
    for cu in (False, True):
        same(call(parts, table, k, v, lens, news, cu), append(parts, k, v, table, lens, news), f"cu={cu}")


@pytest.mark.parametrize("dtype", CODES)
def test_token_by_token_stays_near_the_values(dtype):
    """70 tokens one at a time: each value within half a step of its page's scale for every time that
    the scale grew, plus one (e4m3: a relative 2^-4, or half its smallest step)."""
    H, D, bs, n = 2, 64, 32, 70
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, n, H, D, generator=g).half()
    cache = KVCache.zeros(4, H, D, block=bs, dtype=dtype, device=DEV)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV)
    grown = torch.zeros(4, H, 2)
    for i in range(n):
        before = torch.stack([cache.k_scale.cpu(), cache.v_scale.cpu()], 2)
        kv_append(cache, x[0, i:i + 1].to(DEV), x[1, i:i + 1].to(DEV), table,
                  torch.tensor([i + 1], dtype=torch.int32, device=DEV))
        after = torch.stack([cache.k_scale.cpu(), cache.v_scale.cpu()], 2)
        grown += after > before
    parts = [t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    for h in range(H):
        got = gather(parts, table[0].cpu(), n, h)
        for w in range(2):
            for i in range(n):
                p = int(table[0, i // bs])
                steps, sc = float(grown[p, h, w]) + 1, float(parts[2 + w][p, h])
                want = x[w, i, h].double()
                half = 0.5 * sc if dtype == torch.int8 else torch.maximum(want.abs() * 2.0 ** -4,
                                                                          torch.tensor(sc * 2.0 ** -10))
                assert ((got[w][i] - want).abs() <= steps * half * 1.07 + 1e-9).all(), (h, w, i)


@pytest.mark.parametrize("dtype", CODES)
def test_again_gives_the_same(dtype):
    """An append over its own tokens changes nothing."""
    lens, news = [90, 64], [30, 64]
    parts, table, k, v = problem(2, 128, 64, dtype, lens, news, 11)
    cache = call(parts, table, k, v, lens, news)
    once = [t.cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    kv_append(cache, k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
              offsets(news).to(DEV))
    same(cache, once)


@pytest.mark.parametrize("dtype", CODES)
def test_strides_and_alignment(dtype):
    """Slices of a fused projection's output, at odd offsets and strides, and a strided last dimension."""
    H, D, bs = 2, 64, 16
    lens, news = [20, 33], [20, 7]
    parts, table, k, v = problem(H, D, bs, dtype, lens, news, 13)
    want = append(parts, k, v, table, lens, news)
    n = sum(news)
    for pad, off in ((0, 0), (3, 1), (8, 8)):
        wide = torch.zeros(n, 2 * H * D + 2 * pad, dtype=k.dtype, device=DEV)
        kk, vv = wide[:, off:off + H * D].view(n, H, D), wide[:, off + H * D:off + 2 * H * D].view(n, H, D)
        kk.copy_(k), vv.copy_(v)
        same(call(parts, table, kk, vv, lens, news), want, f"pad {pad}")
    by_d = torch.empty(n, D, H, dtype=k.dtype, device=DEV).transpose(1, 2)
    by_d.copy_(k)
    same(call(parts, table, by_d, v, lens, news), want, "strided values")


@pytest.mark.parametrize("dtype", CODES)
def test_zeros_tiny_and_non_finite(dtype):
    H, D, bs = 1, 64, 16
    lens, news = [16, 20, 16, 16, 18], [16, 4, 16, 16, 2]
    parts, table, k, v = problem(H, D, bs, dtype, lens, news, 17, torch.bfloat16)
    at = offsets(news).tolist()
    k[at[0]:at[1]] = 0
    v[at[1]:at[2]] = 1e-30
    k[at[2] + 3, 0, 5] = math.inf
    v[at[3] + 1, 0, 63] = math.nan
    k[at[4], 0, 1] = -math.inf
    cache = call(parts, table, k, v, lens, news)
    same(cache, append(parts, k, v, table, lens, news))
    assert cache.k_scale[int(table[0, 0]), 0] == 2.0 ** -64
    assert torch.isinf(cache.k_scale[int(table[2, 0]), 0]) and torch.isnan(cache.v_scale[int(table[3, 0]), 0])


def test_no_tokens_pages_out_of_range_and_short_lengths():
    """Sequences without tokens, a table that names no page, tokens past the table, lengths below the
    number of tokens and tokens past the last sequence: nothing else is touched."""
    H, D, bs = 2, 64, 16
    lens, news = [40, 5, 16, 3, 0], [8, 0, 16, 5, 2]
    parts, table, k, v = problem(H, D, bs, torch.int8, [64, 16, 16, 16, 16], news, 19)
    table[2, 0] = 10 ** 6
    table[0, 2] = -5
    k, v = (torch.cat([t, t[:3]]) for t in (k, v))              # three tokens past cu[-1]
    want = append(parts, k, v, table, lens, news)
    same(call(parts, table, k, v, lens, news), want)
    narrow = table[:, :1].contiguous()
    same(call(parts, narrow, k, v, [24, 5, 16, 3, 0], news), append(parts, k, v, narrow, [24, 5, 16, 3, 0], news))
    cache = device_cache(parts)
    none = torch.empty(0, H, D, dtype=torch.float16, device=DEV)
    kv_append(cache, none, none, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
              torch.zeros(6, dtype=torch.int32, device=DEV))
    same(cache, parts)


def test_many_sequences():
    """More sequences than a wavefront looks at in one step."""
    g = torch.Generator().manual_seed(2)
    news = torch.randint(0, 6, (300,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 40, (300,), generator=g))]
    parts, table, k, v = problem(1, 64, 16, torch.int8, lens, news, 23)
    same(call(parts, table, k, v, lens, news), append(parts, k, v, table, lens, news))


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,D,bs", [(2, 128, 64), (1, 64, 16), (1, 256, 128), (2, 192, 32)])
def test_read(H, D, bs, dtype, out):
    g = torch.Generator().manual_seed(bs)
    lens, news = [1, bs, 2 * bs + 7, 5, 3 * bs, 2], [1, bs, bs + 9, 0, 1, 4]      # the last: two before its start
    pages = 12
    parts = random_cache(pages, H, bs, D, dtype, g)
    table = tables(lens, bs, pages, g)
    table[4, 2] = -1
    n, extra = sum(news), 3
    k, v = kv_read(device_cache(parts), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                   offsets(news).to(DEV), total=n + extra, dtype=out)
    at = 0
    for b, m in enumerate(news):
        for h in range(H):
            K, V, _ = gather([t if i < 2 else t for i, t in enumerate(parts)], table[b], lens[b], h)
            pad = max(0, m - lens[b])
            for got, full in ((k, K), (v, V)):
                want = torch.cat([torch.zeros(pad, D, dtype=torch.float64), full[lens[b] - m + pad:]])
                # code * scale of a float32 scale is exact in 64 bits; rounded to float32, then to `out`
                assert torch.equal(got[at:at + m, h].cpu(), want.float().to(out)), (b, h)
        at += m
    assert not k[n:].any() and not v[n:].any()


def test_read_one_token_each():
    g = torch.Generator().manual_seed(1)
    parts = random_cache(6, 2, 16, 64, torch.int8, g)
    table = tables([17, 3], 16, 6, g)
    k, v = kv_read(device_cache(parts), table.to(DEV), torch.tensor([17, 3], dtype=torch.int32, device=DEV))
    for b, L in enumerate((17, 3)):
        K, V, _ = gather(parts, table[b], L, 1)
        assert torch.equal(k[b, 1].cpu(), K[-1].float().half()) and torch.equal(v[b, 1].cpu(), V[-1].float().half())


def test_append_and_read_in_a_graph_and_on_another_stream():
    lens, news = [90, 64], [30, 64]
    parts, table, k, v = problem(2, 128, 64, torch.int8, lens, news, 29)
    want = append(parts, k, v, table, lens, news)
    cache = device_cache(parts)
    first = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    args = (k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
            offsets(news).to(DEV))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        kv_append(cache, *args)
    side.synchronize()
    same(cache, want, "stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_append(cache, *args)
        got = kv_read(cache, *args[2:], total=sum(news))
    eager = kv_read(cache, *args[2:], total=sum(news))
    for _ in range(3):
        for t, f in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), first):
            t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        same(cache, want, "graph")
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def negated(x):
    """A dense view of ``x``'s values whose memory holds -x."""
    y = torch._neg_view(-x)
    assert y.is_neg() and y.stride() == x.stride() and torch.equal(y, x)
    return y


def test_views_that_negate():
    lens, news = [20, 33], [20, 7]
    parts, table, k, v = problem(2, 64, 16, torch.int8, lens, news, 37)
    want = append(parts, k, v, table, lens, news)
    same(call(parts, table, negated(k.to(DEV)), negated(v.to(DEV)), lens, news), want)
    same(call(parts, table, k, negated(v.to(DEV)), lens, news), want)
    on = [t.to(DEV) for t in parts]
    with pytest.raises(ValueError):
        KVCache(on[0], on[1], torch._neg_view(on[2]), on[3])


def test_refusals():
    g = torch.Generator().manual_seed(0)
    parts = [t.to(DEV) for t in random_cache(2, 2, 16, 64, torch.int8, g)]
    cache = KVCache(*parts)
    with pytest.raises(TypeError):
        KVCache(parts[0].float(), *parts[1:])
    with pytest.raises(ValueError):
        KVCache(parts[0], parts[0], *parts[2:])                 # values not transposed
    with pytest.raises(ValueError):
        KVCache(parts[0][:, :, :8], parts[1][..., :8], *parts[2:])
    with pytest.raises(ValueError):
        KVCache(parts[0], parts[1], parts[2][:1], parts[3])
    with pytest.raises(ValueError):
        KVCache(parts[0].cpu(), *parts[1:])
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    x = torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(TypeError):
        kv_append(cache, x.float(), x.float(), table, lens)
    with pytest.raises(ValueError):
        kv_append(cache, x, x[:1], table, lens)
    with pytest.raises(ValueError):
        kv_append(cache, x[:, :1], x[:, :1], table, lens)       # one head of two
    with pytest.raises(ValueError):
        kv_append(cache, x[:1], x[:1], table, lens)             # one token, two sequences, no cu
    with pytest.raises(TypeError):
        kv_append(cache, x, x, table.long(), lens)
    with pytest.raises(ValueError):
        kv_append(cache, x, x, table, lens[:1])
    with pytest.raises(TypeError):
        kv_append(cache, x, x, table, lens, torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        kv_append(cache, x, x, table.cpu(), lens)
    with pytest.raises(ValueError):
        kv_read(cache, table, lens, torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        kv_read(cache, table, lens, dtype=torch.float64)
    with pytest.raises(TypeError):
        kv_append(parts, x, x, table, lens)
