"""kv_rotate_append into the 8-bit cache: against kv_append of keys turned in 64 bits."""
import pytest
import torch

from polar_pack_amd.kv_cache import kv_append, kv_read, kv_rotate_append
from polar_pack_amd.rotary import Rotary, rotate
from serving import DEV, QMAX, device_cache, offsets, random_cache, raw, tables
from serving4 import partners, turn

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
CODES = [torch.int8, torch.float8_e4m3fn]


def problem(H, D, bs, dtype, lens, news, seed, value):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(n, 0) // bs) for n in lens) + 2
    parts = random_cache(pages, H, bs, D, dtype, g)
    k, v = (torch.randn(sum(news), H, D, generator=g).to(value) for _ in range(2))
    return parts, tables(lens, bs, pages, g), k, v, torch.randn(sum(news), 3 * H, D, generator=g).to(value)


def at(table, lens, news, cu=True):
    return (table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), offsets(news).to(DEV) if cu else None)


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("value,pairs", [(F16, "halves"), (BF16, "neighbours")])
@pytest.mark.parametrize("H,D,bs,rot", [(2, 128, 64, 128), (1, 64, 16, 32), (3, 256, 128, 256), (2, 192, 32, 96), (2, 192, 128, 192),
                                        (17, 64, 64, 64), (2, 128, 32, 80)])
def test_turned_append(H, D, bs, rot, value, pairs, dtype):
    """Values and their pages are kv_append's bytes; keys are the turned ones to half a step of the page's scale (e4m3:
    a relative 2^-4, or half a smallest step) and the rotation's own error.  The last includes pages whose old codes
    are rounded again: kv_append's rule, checked by what is read back of tokens that were there."""
    lens, news = [1, bs, bs + 1, 3 * bs - 1, 2 * bs + 5, 7], [1, bs, 2, 2 * bs + 3, 5, 0]
    parts, table, k, v, q = problem(H, D, bs, dtype, lens, news, D + bs + rot, value)
    freqs = [5000.0 ** (-2 * f / rot) for f in range(rot // 2)]
    own = [p for L, n in zip(lens, news) for p in range(L - n, L)]
    cache, plain = device_cache(parts), device_cache(parts)
    r = Rotary(D, base=5000.0, rotary_dim=rot, pairs=pairs)
    where = at(table, lens, news)
    got = kv_rotate_append(cache, q.to(DEV), k.to(DEV), v.to(DEV), r, *where)
    assert torch.equal(got, rotate(q.to(DEV), r, torch.tensor(own, device=DEV)))
    turned = turn(k.double(), rot, pairs, freqs, [0] * (rot // 2), [own])
    kv_append(plain, turned.to(value).to(DEV), v.to(DEV), *where)
    for name in ("v", "v_scale"):
        assert torch.equal(raw(getattr(cache, name)), raw(getattr(plain, name))), name
    rk, _ = kv_read(cache, *where, total=sum(news), dtype=torch.float32)
    # each token's page scale
    seq = [b for b, n in enumerate(news) for _ in range(n)]
    scale = torch.stack([cache.k_scale[int(table[b, p // bs])] for b, p in zip(seq, own)]).cpu().double()[:, :, None]
    off = 2.0 ** -22 * partners(k.double(), rot, pairs) + 2.0 ** -22 * turned.abs()
    step = 0.5 * scale if dtype == torch.int8 else torch.maximum(2.0 ** -4 * turned.abs(), 2.0 ** -10 * scale)
    assert ((rk.cpu().double() - turned).abs() <= step * (1 + 2.0 ** -20) + off).all()
    # no page's scale is larger than what its values ask for, within the rounding of keys to 16 bits
    ratio = cache.k_scale / plain.k_scale
    assert (ratio - 1).abs().max() <= torch.finfo(value).eps
    before, _ = kv_read(plain, *at(table, [L - n for L, n in zip(lens, news)], [min(L - n, bs) for L, n in zip(lens, news)]),
                        total=sum(min(L - n, bs) for L, n in zip(lens, news)), dtype=torch.float32)
    after, _ = kv_read(cache, *at(table, [L - n for L, n in zip(lens, news)], [min(L - n, bs) for L, n in zip(lens, news)]),
                       total=sum(min(L - n, bs) for L, n in zip(lens, news)), dtype=torch.float32)
    top = float(cache.k_scale.max()) * QMAX[dtype]
    assert ((after - before).abs() <= top * (2.0 / 127 if dtype == torch.int8 else 2.0 ** -3)).all()


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("wide", [True, False])
def test_given_positions_are_those_of_rotate(dtype, wide):
    """Positions that turn nothing leave kv_append's bytes; others the bytes of the same turned another way round."""
    lens, news = [50, 20], [33, 20]
    parts, table, k, v, q = problem(2, 128, 16, dtype, lens, news, 11, F16)
    where, r = at(table, lens, news), Rotary(128, sections=(16, 24, 24))
    cache, plain = device_cache(parts), device_cache(parts)
    none = torch.zeros(3, 53, dtype=torch.int64 if wide else torch.int32, device=DEV)
    got = kv_rotate_append(cache, q.to(DEV), k.to(DEV), v.to(DEV), r, *where, positions=none)
    kv_append(plain, k.to(DEV), v.to(DEV), *where)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(raw(getattr(cache, name)), raw(getattr(plain, name))), name
    assert torch.equal(got.cpu(), q)
    own = torch.cat([torch.arange(17, 50), torch.arange(20)]).to(DEV)
    one, two = device_cache(parts), device_cache(parts)
    a = kv_rotate_append(one, q.to(DEV), k.to(DEV), v.to(DEV), r, *where)
    b = kv_rotate_append(two, q.to(DEV), k.to(DEV), v.to(DEV), r, *where, positions=own.to(none.dtype).expand(3, 53))
    assert torch.equal(a, b)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(raw(getattr(one, name)), raw(getattr(two, name))), name


def test_single_tokens_and_tokens_of_no_sequence():
    lens = [1, 16, 17, 33, 400]
    parts, table, k, v, q = problem(2, 64, 16, torch.int8, lens, [1] * 5, 3, BF16)
    r = Rotary(64)
    cache, other = device_cache(parts), device_cache(parts)
    got = kv_rotate_append(cache, q.to(DEV), k.to(DEV), v.to(DEV), r, *at(table, lens, [1] * 5, cu=False))
    more = [torch.cat([x, torch.ones(2, *x.shape[1:], dtype=BF16)]).to(DEV) for x in (q, k, v)]
    same = kv_rotate_append(other, *more, r, *at(table, lens, [1] * 5))
    assert torch.equal(same[:5], got) and not same[5:].any()
    assert torch.equal(cache.k, other.k) and torch.equal(cache.k_scale, other.k_scale)
    own = torch.tensor(lens, device=DEV) - 1
    assert torch.equal(got, rotate(q.to(DEV), r, own))
    kept = device_cache(parts)                                # given positions turn every row
    pos = torch.arange(7, device=DEV)
    assert torch.equal(kv_rotate_append(kept, *more, r, *at(table, lens, [1] * 5), positions=pos), rotate(more[0], r, pos))


def test_empty_sequences_between():
    """Queries find their sequence among many without tokens."""
    news = [0] * 130 + [3] + [0] * 70 + [40, 0, 1]
    lens = [5] * 130 + [9] + [0] * 70 + [40, 8, 100]
    parts, table, k, v, q = problem(1, 64, 16, torch.int8, lens, news, 5, F16)
    own = torch.tensor([p for L, n in zip(lens, news) for p in range(L - n, L)], device=DEV)
    r = Rotary(64)
    got = kv_rotate_append(device_cache(parts), q.to(DEV), k.to(DEV), v.to(DEV), r, *at(table, lens, news))
    assert torch.equal(got, rotate(q.to(DEV), r, own))


def test_keys_that_are_not_finite():
    parts, table, k, v, q = problem(2, 64, 16, torch.int8, [20], [20], 6, F16)
    k[18, 1, 5] = float("inf")
    cache = device_cache(parts)
    kv_rotate_append(cache, None, k.to(DEV), v.to(DEV), Rotary(64), *at(table, [20], [20]))
    scales = cache.k_scale.cpu()[table[0, :2].long()]
    assert torch.isfinite(scales).tolist() == [[True, True], [True, False]]
    assert torch.isfinite(cache.v_scale).all()


@pytest.mark.parametrize("stream", [False, True])
def test_capture(stream):
    parts, table, k, v, q = problem(2, 128, 64, torch.int8, [300, 200], [1, 1], 7, F16)
    r, lens, t = Rotary(128), torch.tensor([101, 63], dtype=torch.int32, device=DEV), table.to(DEV)
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    cache, eager = device_cache(parts), device_cache(parts)
    kv_rotate_append(device_cache(parts), q, k, v, r, t, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_rotate_append(cache, q, k, v, r, t, lens)
    for step in range(4):
        lens.add_(1)
        for x in (q, k, v):
            x.normal_()
        side = torch.cuda.Stream() if stream else torch.cuda.current_stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = kv_rotate_append(eager, q, k, v, r, t, lens)
        torch.cuda.current_stream().wait_stream(side)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v) and torch.equal(cache.k_scale, eager.k_scale)
