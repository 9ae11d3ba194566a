"""kv_rotate_append and rotate where the first tests of them do not look: operands at odd places, more than four axes."""
import pytest
import torch

from polar_pack_amd.kv_cache import kv_append, kv_rotate_append
from polar_pack_amd.rotary import Rotary, rotate
from serving import DEV, device_cache, offsets, random_cache, raw, tables
from serving4 import append4, device_cache4, partners, random_cache4, turn
from test_gpu_kv_cache4 import same
from test_gpu_rotary import check

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
NAMES = ("k", "v", "k_scale", "v_scale")
KINDS = [torch.int8, torch.float8_e4m3fn, "4 bits"]


def caches(kind, pages, H, bs, D, g):
    parts = random_cache4(pages, H, bs, D, g) if kind == "4 bits" else random_cache(pages, H, bs, D, kind, g)
    make = device_cache4 if kind == "4 bits" else device_cache
    return lambda: make(parts)


def places(x):
    """The same (tokens, heads, D) values at other places: behind one value, in rows of odd lengths, heads before tokens, a
    row's values apart, held negated."""
    T, H, D = x.shape
    room = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    yield "one value on", room[1:].view(T, H, D).copy_(x)
    wide = torch.zeros(T, H + 1, D + 3, dtype=x.dtype, device=x.device)
    wide[:, :H, :D] = x
    yield "rows of odd lengths", wide[:, :H, :D]
    yield "heads before tokens", x.transpose(0, 1).contiguous().transpose(0, 1)
    yield "values apart", x.transpose(1, 2).contiguous().transpose(1, 2)
    yield "negated", torch._neg_view(-x)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("value", [F16, BF16])
@pytest.mark.parametrize("H,Hq,D,bs,rot,pairs", [(2, 5, 64, 16, 64, "halves"), (3, 12, 128, 64, 96, "neighbours"), (1, 7, 192, 32, 192, "halves"),
                                                 (2, 2, 256, 128, 256, "neighbours")])
@pytest.mark.parametrize("given", [True, False])
def test_odd_places(H, Hq, D, bs, rot, pairs, value, kind, given):
    """Wherever queries, keys and values lie, the cache's bytes and the queries are those of dense ones."""
    lens, news = [1, 2 * bs + 5, 40, 7], [1, bs + 9, 3, 0]
    g = torch.Generator().manual_seed(D + bs)
    pages = sum(-(-n // bs) for n in lens) + 1
    fresh = caches(kind, pages, H, bs, D, g)
    table, n = tables(lens, bs, pages, g).to(DEV), sum(news)
    at = (table, torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV))
    q, k, v = (torch.randn(n, h, D, generator=g).to(value).to(DEV) for h in (Hq, H, H))
    r = Rotary(D, rotary_dim=rot, pairs=pairs)
    pos = torch.randint(0, 10 ** 5, (n,), generator=g).to(DEV) if given else None
    dense = fresh()
    want = kv_rotate_append(dense, q, k, v, r, *at, positions=pos)
    if given:
        assert torch.equal(want, rotate(q, r, pos))
    for (name, oq), (_, ok), (_, ov) in zip(places(q), places(k), places(v)):
        for args in ((oq, ok, ov), (oq, k, v), (q, ok, v), (q, k, ov)):
            cache = fresh()
            assert torch.equal(kv_rotate_append(cache, *args, r, *at, positions=pos), want), name
            for part in NAMES:
                assert torch.equal(raw(getattr(cache, part)), raw(getattr(dense, part))), (name, part)


@pytest.mark.parametrize("kind", KINDS)
def test_single_tokens_at_odd_places(kind):
    lens = [1, 16, 17, 33, 400]
    g = torch.Generator().manual_seed(8)
    fresh = caches(kind, 34, 2, 16, 64, g)
    table, at_len = tables(lens, 16, 34, g).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(5, h, 64, generator=g).half().to(DEV) for h in (9, 2, 2))
    r, dense = Rotary(64), fresh()
    want = kv_rotate_append(dense, q, k, v, r, table, at_len)
    for (name, oq), (_, ok), (_, ov) in zip(places(q), places(k), places(v)):
        cache = fresh()
        assert torch.equal(kv_rotate_append(cache, oq, ok, ov, r, table, at_len), want), name
        for part in NAMES:
            assert torch.equal(raw(getattr(cache, part)), raw(getattr(dense, part))), (name, part)


def several(n_axes, n):
    """Axes in turn, some of them turning nothing."""
    return [(7 * i) % n_axes for i in range(n)]


@pytest.mark.parametrize("n_axes", [5, 6, 64, 255])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("wide", [True, False])
def test_rotate_of_many_axes(n_axes, wide, pairs):
    g = torch.Generator().manual_seed(n_axes)
    x = torch.randn(21, 3, 128, generator=g).bfloat16()
    pos = torch.randint(-5000, 50000, (n_axes, 21), generator=g)
    axes = several(n_axes, 64)
    axes[0] = n_axes - 1
    freqs = [0.9 ** f for f in range(64)]
    r = Rotary(128, inv_freq=freqs, pairs=pairs, axes=axes)
    assert r.n_axes == n_axes
    got = rotate(x.to(DEV), r, (pos if wide else pos.int()).to(DEV))
    check(x, got, turn(x.double(), 128, pairs, freqs, axes, pos.tolist()), 128, pairs)


@pytest.mark.parametrize("n_axes", [5, 64])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_append_of_many_axes(n_axes, pairs):
    """4 bits, byte for byte; in 8 bits the values, and the keys to half a step and the rotation's error; queries as rotate."""
    H, D, bs, lens, news = 2, 128, 32, [50, 33], [37, 33]
    g = torch.Generator().manual_seed(n_axes)
    parts, table = random_cache4(5, H, bs, D, g), tables(lens, bs, 5, g)
    n = sum(news)
    q, k, v = (torch.randn(n, h, D, generator=g).half() for h in (6, H, H))
    pos, axes = torch.randint(0, 30000, (n_axes, n), generator=g), several(n_axes, 64)
    axes[5] = n_axes - 1
    freqs = [0.8 ** f for f in range(64)]
    r = Rotary(D, inv_freq=freqs, pairs=pairs, axes=axes)
    at = (table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV))
    turned = turn(k.double(), D, pairs, freqs, axes, pos.tolist())
    cache = device_cache4(parts)
    got = kv_rotate_append(cache, q.to(DEV), k.to(DEV), v.to(DEV), r, *at, positions=pos.to(DEV))
    assert torch.equal(got, rotate(q.to(DEV), r, pos.to(DEV)))
    same(cache, append4(parts, turned, v.double(), table, lens, news))
    parts8 = random_cache(5, H, bs, D, torch.int8, g)
    eight, plain = device_cache(parts8), device_cache(parts8)
    assert torch.equal(kv_rotate_append(eight, q.to(DEV), k.to(DEV), v.to(DEV), r, *at, positions=pos.int().to(DEV)), got)
    kv_append(plain, k.to(DEV), v.to(DEV), *at)
    assert torch.equal(eight.v, plain.v) and torch.equal(eight.v_scale, plain.v_scale)
    off = 2.0 ** -22 * (partners(k.double(), D, pairs) + turned.abs())
    i = 0
    for b, m in enumerate(news):
        for p in range(lens[b] - m, lens[b]):
            page = int(table[b, p // bs])
            s = eight.k_scale[page].cpu().double()[:, None]
            read = eight.k[page, :, p % bs].cpu().double() * s
            assert ((read - turned[i]).abs() <= 0.5 * s * (1 + 2.0 ** -20) + off[i]).all()
            i += 1


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("H,D,bs", [(2, 128, 64), (1, 64, 16), (1, 256, 128)])
def test_codes_that_are_rounded_again(H, D, bs, kind):
    """Where a page's scale grew, its earlier tokens' codes are round(code * (old / new)) of the scales before and after, to
    the bit; where it did not, they are as they were; and the new scale is what the turned keys ask for, to their own error."""
    lens, news = [bs - 1, 2 * bs - 3, bs + 9, 3 * bs - 5], [2, 7, 5, bs]
    g = torch.Generator().manual_seed(D)
    pages = sum(-(-n // bs) for n in lens)
    parts, table = random_cache(pages, H, bs, D, kind, g), tables(lens, bs, pages, g)
    k, v = (torch.randn(sum(news), H, D, generator=g).half() for _ in range(2))
    k[2:9] *= 0.02                                               # a page whose scale stays
    cache = device_cache(parts)
    freqs = [10000.0 ** (-2 * f / D) for f in range(D // 2)]
    at = (table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV))
    kv_rotate_append(cache, None, k.to(DEV), v.to(DEV), Rotary(D), *at)
    own = [p for L, n in zip(lens, news) for p in range(L - n, L)]
    turned = turn(k.double(), D, "halves", freqs, [0] * (D // 2), [own])
    pair = partners(k.double(), D, "halves")
    now, was = cache.k_scale.cpu(), parts[2]
    qmax = 127.0 if kind == torch.int8 else 448.0
    grew = kept = i = 0
    for b, (L, n) in enumerate(zip(lens, news)):
        first = (L - n) // bs                                    # the page that holds earlier tokens
        page, held, new = int(table[b, first]), (L - n) % bs, min(n, bs - (L - n) % bs)
        top = turned[i:i + new].abs().amax((0, 2))
        off = pair[i:i + new].amax((0, 2)) * 2.0 ** -22
        i += n
        if held == 0:
            continue
        for h in range(H):
            need = torch.clamp(top[h] / qmax, min=float(was[page, h]))
            assert abs(float(now[page, h]) - float(need)) <= float(off[h]) / qmax + 2.0 ** -23 * float(need)
            old = parts[0][page, h, :held]
            if now[page, h] > was[page, h]:
                x = old.float() * (was[page, h] / now[page, h])
                old = (x.round() if kind == torch.int8 else x).to(kind)
                grew += 1
            else:
                assert now[page, h] == was[page, h]
                kept += 1
            assert torch.equal(raw(cache.k[page, h, :held]).cpu(), raw(old))
    assert grew and kept
