"""kv_append, kv_rotate_append and kv_read of the 4-bit cache: codes and scales against the 64-bit definition bit for
bit (both are exact functions of the values; turned keys differ from the 64-bit form's by 2^-50, so that one in some
10^13 could fall on the other side of a border)."""
import math

import pytest
import torch

from polar_pack_amd.kv_cache import KVCache4, kv_append, kv_read, kv_rotate_append
from polar_pack_amd.rotary import Rotary, rotate
from serving import DEV, offsets, tables
from serving4 import append4, device_cache4, f8, plain_parts, random_cache4, turn, unpack, value4

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
NAMES = ("k", "v", "k_scale", "v_scale")
SHAPES = [(2, 128, 64), (1, 64, 16), (3, 256, 128), (2, 192, 32), (1, 192, 16)]


def same(cache, want, ctx=""):
    """Byte for byte, but for the codes of tokens that are marked as not finite, which are open."""
    got = [getattr(cache, name).cpu() for name in NAMES]
    marked = f8(want[2]).isnan().any(-1)                                   # (pages, H, block)
    H, bs = marked.shape[1:]
    for name, x, w in zip(NAMES, got, want):
        x, w = x.view(torch.uint8), w.view(torch.uint8)
        if name == "k":
            off = (x != w) & ~marked[..., None]
        elif name == "k_scale":
            off = x != w
        elif name == "v":
            off = (unpack(x) != unpack(w)) & ~marked[:, :, None]
        else:
            off = (x != w) & ~marked[:, :, None]
        count = int(off.sum())
        assert count == 0, f"{ctx} {name}: {count} differ, the first at {off.nonzero()[0].tolist()}"


def problem(H, D, bs, lens, news, seed, value=F16, size=1.0):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(n, 0) // bs) for n in lens) + 2
    parts = random_cache4(pages, H, bs, D, g)
    table = tables(lens, bs, pages, g)
    spread = torch.exp(torch.randn(H, D, generator=g)) * size
    k, v = ((torch.randn(sum(news), H, D, generator=g) * spread).to(value) for _ in range(2))
    return parts, table, k, v


def at(table, lens, news, cu=True):
    return (table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV) if cu else None)


@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("H,D,bs", SHAPES)
def test_append_matches_the_definition(H, D, bs, value):
    """Pages begun, filled, gone on with at even and odd places; everything else stays as it was."""
    lens, news = [1, bs, bs + 1, 3 * bs - 1, 2 * bs + 5, 7], [1, bs, 2, 2 * bs + 3, 5, 0]
    parts, table, k, v = problem(H, D, bs, lens, news, D + bs, value)
    cache = device_cache4(parts)
    kv_append(cache, k.to(DEV), v.to(DEV), *at(table, lens, news))
    same(cache, append4(parts, k.double(), v.double(), table, lens, news))


@pytest.mark.parametrize("value", [F16, BF16])
def test_token_by_token_is_the_same(value):
    """A token's codes depend on no other: one call, or one a token, leaves the same bytes."""
    parts, table, k, v = problem(2, 64, 16, [40, 37], [40, 37], 5, value)
    whole, single = device_cache4(parts), device_cache4(parts)
    kv_append(whole, k.to(DEV), v.to(DEV), *at(table, [40, 37], [40, 37]))
    for i in range(37):
        rows = torch.tensor([i, 40 + i])
        kv_append(single, k[rows].to(DEV), v[rows].to(DEV), *at(table, [i + 1, i + 1], [1, 1], cu=False))
    kv_append(single, k[37:40].to(DEV), v[37:40].to(DEV), *at(table[:1], [40], [3]))
    for name in NAMES:
        assert torch.equal(getattr(whole, name).view(torch.uint8), getattr(single, name).view(torch.uint8)), name


@pytest.mark.parametrize("value,size", [(F16, 1e-4), (F16, 2.0 ** -22), (BF16, 1e-30), (F16, 8000.0), (BF16, 1e5), (BF16, 1e30)])
def test_values_of_any_size(value, size):
    """Below the smallest scale and above the largest: steps of 2^-15, magnitudes held to 6 * 2^13."""
    lens = news = [33]
    parts, table, k, v = problem(2, 128, 64, lens, news, 6, value, size)
    k[3] = 0
    cache = device_cache4(parts)
    kv_append(cache, k.to(DEV), v.to(DEV), *at(table, lens, news))
    same(cache, append4(parts, k.double(), v.double(), table, lens, news))


def test_borders():
    """Values halfway between codes go to the even code, largest ones at and beside 7 scales, zeros of either sign."""
    codes = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    x = torch.cat([codes, codes * (1 + 2.0 ** -10), codes * (1 - 2.0 ** -10)]).half()
    k = torch.zeros(64, 1, 64, dtype=F16)
    for t in range(64):
        k[t, 0, :30] = x * (1 if t % 2 else -1) * 2.0 ** (t // 4 - 8)
        k[t, 0, 31] = torch.tensor([0.0, 7.0, 7.0 * (1 + 2.0 ** -10), 6.9][t % 4]) * 2.0 ** (t // 4 - 8)
        k[t, 0, 32:] = k[t, 0, :32].flip(0) * 0.5
    v = -k.flip(0)
    g = torch.Generator().manual_seed(7)
    parts, table = random_cache4(2, 1, 64, 64, g), torch.tensor([[1]], dtype=torch.int32)
    cache = device_cache4(parts)
    kv_append(cache, k.to(DEV), v.to(DEV), *at(table, [64], [64]))
    want = append4(parts, k.double(), v.double(), table, [64], [64])
    for got, w in zip((cache.k, cache.v), want):                 # the sign of a zero is open
        a, b = unpack(got.cpu()), unpack(w)
        assert torch.equal(value4(a), value4(b))
    for name, w in zip(NAMES[2:], want[2:]):
        assert torch.equal(getattr(cache, name).cpu().view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("H,D,bs", SHAPES)
def test_read(H, D, bs, dtype):
    """Any piece of the tokens, at odd places, from pages that are not there, tokens of no sequence."""
    lens, news = [1, bs, 2 * bs + 7, 3 * bs - 1, 5, 2 * bs], [1, bs - 3, bs + 9, 2, 0, 2 * bs]
    g = torch.Generator().manual_seed(D * bs)
    pages = sum(-(-n // bs) for n in lens) + 2
    parts = random_cache4(pages, H, bs, D, g)
    table = tables(lens, bs, pages, g)
    table[5, 0] = -1
    K, V, _, _ = plain_parts(parts)
    total = sum(news) + 3
    k, v = kv_read(device_cache4(parts), *at(table, lens, news), total=total, dtype=dtype)
    want = torch.zeros(2, total, H, D, dtype=torch.float64)
    i = 0
    for b, n in enumerate(news):
        for pos in range(lens[b] - n, lens[b]):
            p = int(table[b, pos // bs])
            if p >= 0:
                want[0, i], want[1, i] = K[p, :, pos % bs], V[p, :, :, pos % bs]
            i += 1
    for got, w in ((k, want[0]), (v, want[1])):
        assert got.dtype == dtype and torch.equal(got.cpu().double(), w)      # 2 bits times a power of two


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_tokens_that_are_not_finite(what, where, turned):
    """One such value marks its token and head, of keys and of values, and no other."""
    lens = news = [70]
    parts, table, k, v = problem(3, 128, 64, lens, news, 8)
    (k if where == "k" else v)[41, 1, 77] = what
    cache = device_cache4(parts)
    args = (k.to(DEV), v.to(DEV))
    if turned:
        kv_rotate_append(cache, None, *args, Rotary(128), *at(table, lens, news))
    else:
        kv_append(cache, *args, *at(table, lens, news))
    rk, rv = kv_read(cache, *at(table, lens, news), total=70)
    lost = torch.zeros(70, 3, dtype=torch.bool)
    lost[41, 1] = True
    for r in (rk, rv):
        assert torch.equal(r.isnan().cpu(), lost[..., None].expand(70, 3, 128))
    kv_append(cache, *(torch.ones(1, 3, 128, device=DEV).half() for _ in range(2)), *at(table, [42], [1]))
    assert torch.isfinite(kv_read(cache, *at(table, lens, news), total=70)[0]).all()      # written anew


def test_pages_that_are_not_there():
    """Places past the table, pages outside the cache, lengths below the number of tokens: nothing is written."""
    lens, news = [100, 200, 3, 40], [20, 30, 9, 40]
    parts, table, k, v = problem(2, 64, 16, [96, 96, 16, 48], news, 9)
    table = table.clone()
    table[3, 1] = 10 ** 6
    table[0, 5] = -7
    cache = device_cache4(parts)
    extra = torch.randn(5, 2, 64).half()
    kv_append(cache, torch.cat([k, extra]).to(DEV), torch.cat([v, extra]).to(DEV), *at(table, lens, news))
    same(cache, append4(parts, k.double(), v.double(), table, lens, news))


@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("H,D,bs,rot", [(2, 128, 64, 128), (1, 64, 16, 32), (3, 256, 128, 256), (2, 192, 32, 96), (9, 64, 128, 64),
                                        (2, 128, 32, 80)])
def test_turned_append(H, D, bs, rot, pairs, value):
    """At each token's own place: keys turned in 64 bits, queries as rotate turns them."""
    lens, news = [1, bs, bs + 1, 3 * bs - 1, 2 * bs + 5, 7], [1, bs, 2, 2 * bs + 3, 5, 0]
    parts, table, k, v = problem(H, D, bs, lens, news, D + bs + rot, value)
    q = torch.randn(sum(news) + 3, 4 * H, D).to(value)
    kx, vx = (torch.cat([x, torch.ones(3, H, D, dtype=value)]) for x in (k, v))         # tokens of no sequence
    freqs = [5000.0 ** (-2 * f / rot) for f in range(rot // 2)]
    own = [p for L, n in zip(lens, news) for p in range(L - n, L)]
    cache, r = device_cache4(parts), Rotary(D, base=5000.0, rotary_dim=rot, pairs=pairs)
    got = kv_rotate_append(cache, q.to(DEV), kx.to(DEV), vx.to(DEV), r, *at(table, lens, news))
    turned = turn(k.double(), rot, pairs, freqs, [0] * (rot // 2), [own])
    same(cache, append4(parts, turned, v.double(), table, lens, news))
    assert torch.equal(got[:-3], rotate(q[:-3].to(DEV), r, torch.tensor(own, device=DEV)))
    assert not got[-3:].any()
    again = device_cache4(parts)
    assert kv_rotate_append(again, None, kx.to(DEV), vx.to(DEV), r, *at(table, lens, news)) is None
    same(again, [getattr(cache, n).cpu() for n in NAMES])


@pytest.mark.parametrize("wide", [True, False])
def test_turned_append_of_given_positions(wide):
    lens, news = [50, 20], [33, 20]
    parts, table, k, v = problem(2, 128, 16, lens, news, 11, BF16)
    pos = torch.randint(-3000, 10 ** 6, (3, 53), generator=torch.Generator().manual_seed(1))
    r = Rotary(128, sections=(16, 24, 24), scaling=0.5)
    axes = [0] * 16 + [1] * 24 + [2] * 24
    freqs = [10000.0 ** (-f / 64) for f in range(64)]
    q = torch.randn(53, 4, 128).bfloat16().to(DEV)
    p = (pos if wide else pos.int()).to(DEV)
    cache = device_cache4(parts)
    got = kv_rotate_append(cache, q, k.to(DEV), v.to(DEV), r, *at(table, lens, news), positions=p)
    turned = turn(k.double(), 128, "halves", freqs, axes, pos.tolist(), 0.5)
    same(cache, append4(parts, turned, v.double(), table, lens, news))
    assert torch.equal(got, rotate(q, r, p))


def test_single_tokens_of_many_sequences():
    lens = [1 + 37 * i % 130 for i in range(70)]
    parts, table, k, v = problem(2, 64, 16, lens, [1] * 70, 12)
    q = torch.randn(70, 6, 64).half().to(DEV)
    r = Rotary(64)
    cache = device_cache4(parts)
    got = kv_rotate_append(cache, q, k.to(DEV), v.to(DEV), r, *at(table, lens, [1] * 70, cu=False))
    own = [n - 1 for n in lens]
    turned = turn(k.double(), 64, "halves", [10000.0 ** (-f / 32) for f in range(32)], [0] * 32, [own])
    same(cache, append4(parts, turned, v.double(), table, lens, [1] * 70))
    assert torch.equal(got, rotate(q, r, torch.tensor(own, device=DEV)))


def test_slices_and_odd_places():
    """Keys and values as slices of a fused projection, at odd addresses, negated, transposed; a cache that is a slice of
    a larger one, whose neighbours stay."""
    lens, news = [45], [45]
    parts, table, k, v = problem(2, 64, 16, lens, news, 13)
    want = append4(parts, k.double(), v.double(), table, lens, news)
    fused = torch.cat([k, v], 1).to(DEV)
    odd = torch.empty(fused.numel() + 1, dtype=F16, device=DEV)[1:].view(fused.shape).copy_(fused)
    for x in (fused, odd, torch._neg_view(-fused), fused.transpose(0, 2).contiguous().transpose(0, 2)):
        cache = device_cache4(parts)
        kv_append(cache, x[:, :2], x[:, 2:], *at(table, lens, news))
        same(cache, want)
    big = [torch.full((t.shape[0] + 2, *t.shape[1:]), 9, dtype=torch.uint8, device=DEV) for t in parts]
    for b, t in zip(big, parts):
        b[1:-1] = t.view(torch.uint8).to(DEV)
    cache = KVCache4(*[b[1:-1].view(t.dtype) for b, t in zip(big, parts)])
    kv_append(cache, fused[:, :2], fused[:, 2:], *at(table, lens, news))
    same(cache, want)
    assert all((b[0] == 9).all() and (b[-1] == 9).all() for b in big)


def test_capture():
    """A step captured once and replayed as lengths grow, with eager calls on another cache between."""
    parts, table, k, v = problem(2, 128, 16, [90, 90], [1, 1], 14)
    r, lens = Rotary(128), torch.tensor([40, 17], dtype=torch.int32, device=DEV)
    k, v, q = k.to(DEV), v.to(DEV), torch.randn(2, 8, 128, device=DEV).half()
    cache, eager, t = device_cache4(parts), device_cache4(parts), table.to(DEV)
    kv_rotate_append(device_cache4(parts), q, k, v, r, t, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_rotate_append(cache, q, k, v, r, t, lens)
    for step in range(4):
        lens.add_(1 + step)
        for x in (q, k, v):
            x.normal_()
        want = kv_rotate_append(eager, q, k, v, r, t, lens)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        same(cache, [getattr(eager, n).cpu() for n in NAMES], f"step {step}")


def test_refusals():
    c4 = KVCache4.zeros(4, 2, 64, block=16)
    k = torch.zeros(3, 2, 64, device=DEV).half()
    q, r = torch.zeros(3, 4, 64, device=DEV).half(), Rotary(64)
    t, lens, cu = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV), offsets([3]).to(DEV)
    for bad, exc in ((lambda: kv_rotate_append(c4, q[:2], k, k, r, t, lens, cu), ValueError),
                     (lambda: kv_rotate_append(c4, q.bfloat16(), k, k, r, t, lens, cu), ValueError),
                     (lambda: kv_rotate_append(c4, q, k, k[:2], r, t, lens, cu), ValueError),
                     (lambda: kv_rotate_append(c4, q, k, k, None, t, lens, cu), TypeError),
                     (lambda: kv_rotate_append(c4, q, k, k, Rotary(128), t, lens, cu), ValueError),
                     (lambda: kv_rotate_append(c4, q, k, k, Rotary(64, sections=(16, 16)), t, lens, cu, positions=lens), ValueError),
                     (lambda: kv_rotate_append(c4, q, k, k, r, t, lens, cu, positions=torch.zeros(2, dtype=torch.int32, device=DEV)), ValueError),
                     (lambda: kv_rotate_append(c4, q, k, k, r, t, lens, cu, positions=torch.zeros(3, device=DEV)), TypeError),
                     (lambda: kv_rotate_append(c4, q, k, k, r, t, lens), ValueError),
                     (lambda: kv_rotate_append(None, q, k, k, r, t, lens, cu), TypeError),
                     (lambda: kv_append(c4, k.float(), k.float(), t, lens, cu), TypeError),
                     (lambda: KVCache4(c4.k.int(), c4.v, c4.k_scale, c4.v_scale), TypeError),
                     (lambda: KVCache4(c4.k, c4.v[:, :, :32], c4.k_scale, c4.v_scale), ValueError),
                     (lambda: KVCache4(c4.k, c4.v, c4.v_scale, c4.k_scale), ValueError),
                     (lambda: KVCache4(c4.k, c4.v, c4.k_scale.view(torch.uint8), c4.v_scale), ValueError),
                     (lambda: KVCache4(c4.k[:, :1], c4.v[:, :1], c4.k_scale[:, :1], c4.v_scale[:, :1]), ValueError),
                     (lambda: KVCache4(c4.k.cpu(), c4.v, c4.k_scale, c4.v_scale), ValueError),
                     (lambda: KVCache4.zeros(4, 2, 80), ValueError), (lambda: KVCache4.zeros(4, 2, 64, block=48), ValueError)):
        with pytest.raises(exc):
            bad()
    assert not c4.k.any() and not c4.v.any()
    none = torch.zeros(0, 2, 64, device=DEV).half()
    empty = kv_rotate_append(c4, none, none, none, r, t, lens, offsets([0]).to(DEV))
    assert empty.shape == (0, 2, 64)
