"""rotate against 64-bit rotations whose angles are reduced in whole numbers, element by element.

The bound: sines and cosines are off by at most 2^-23 (their series in float32 and a 2^-32 of a turn), the two
products and their sum by 2^-24 of |a| + |b| each, the factor `scaling` by 2^-24 once more, so 2^-22 of
scaling * (|a| + |b|) holds with room; then one rounding to the type."""
import pytest
import torch

from polar_pack_amd.rotary import Rotary, rotate
from serving import DEV
from serving4 import partners, turn

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def check(x, got, want, rot, pairs, scaling=1.0):
    eps = torch.finfo(x.dtype).eps / 2
    tol = 2.0 ** -22 * abs(scaling) * partners(x.double(), rot, pairs) + eps * want.abs() + torch.finfo(x.dtype).tiny * eps
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.cpu().double() - want).abs() / tol.clamp(min=1e-30)).max()))
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("T,heads,D,rot", [(1, 1, 16, 16), (5, 3, 64, 64), (33, 2, 80, 80), (3, 18, 128, 128), (7, 5, 128, 48),
                                           (300, 3, 96, 32), (9, 1, 512, 512), (4, 7, 72, 64), (2, 3, 24, 16), (130, 2, 256, 240)])
def test_one_axis(T, heads, D, rot, pairs, dtype):
    g = torch.Generator().manual_seed(T + D)
    x = (torch.randn(T, heads, D, generator=g) * 3).to(dtype)
    pos = torch.randint(-5000, 140000, (T,), generator=g)
    pos[0] = 0
    freqs = [10000.0 ** (-2 * f / rot) for f in range(rot // 2)]
    want = turn(x.double(), rot, pairs, freqs, [0] * (rot // 2), [pos.tolist()])
    r = Rotary(D, rotary_dim=rot, pairs=pairs)
    got = rotate(x.to(DEV), r, pos.to(DEV))
    check(x, got, want, rot, pairs)
    assert torch.equal(got[0].cpu(), x[0])                    # position 0 turns nothing
    assert torch.equal(rotate(x.to(DEV), r, pos.int().to(DEV)), got)
    assert torch.equal(rotate(x.to(DEV), r, pos[None].to(DEV)), got)


@pytest.mark.parametrize("T,heads", [(1, 1), (1, 70), (40000, 1), (3, 40), (1000, 33)])
def test_token_and_head_counts(T, heads):
    """Every split of heads over threads: against rows turned one call a head."""
    x = torch.randn(T, heads, 64, device=DEV).half()
    pos = torch.randint(0, 10 ** 6, (T,), device=DEV)
    r = Rotary(64)
    whole = rotate(x, r, pos)
    for h in {0, heads // 2, heads - 1}:
        assert torch.equal(whole[:, h:h + 1], rotate(x[:, h:h + 1], r, pos))


@pytest.mark.parametrize("pos", [2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345, -2 ** 53 - 7, 2 ** 62, 1])
def test_far_positions(pos):
    """Angles keep all their bits: the frequency is held to 2^-65 of a turn, so that is what the position multiplies."""
    x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(1))
    freqs = [10000.0 ** (-f / 32) for f in range(32)]
    want = turn(x.double(), 64, "halves", freqs, [0] * 32, [[pos]])
    got = rotate(x.to(DEV), Rotary(64), torch.tensor([pos], device=DEV)).cpu().double()
    tol = 2.0 ** -22 * partners(x.double(), 64, "halves") + 2.0 ** -24 * want.abs()
    tol += abs(pos) * 2.0 ** -65 * 6.3 * partners(x.double(), 64, "halves")
    assert ((got - want).abs() <= tol).all()


def test_turning_back():
    x = torch.randn(50, 3, 128, device=DEV)
    pos = torch.randint(0, 10 ** 7, (50,), device=DEV)
    r = Rotary(128)
    back = rotate(rotate(x, r, pos), r, -pos)
    # two rotations, each within 2^-22 of the pair and one rounding
    pair = (x[..., :64].abs() + x[..., 64:].abs()).repeat(1, 1, 2)
    assert ((back - x).abs() <= 2.0 ** -20 * pair).all()


@pytest.mark.parametrize("kind", ["sections", "axes", "empty"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("wide", [True, False])
def test_axes(kind, pairs, wide):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 5, 128, generator=g).bfloat16()
    n_axes = 4 if kind == "empty" else 3
    pos = torch.randint(0, 9000, (n_axes, 40), generator=g)
    args = {"sections": dict(sections=(16, 24, 24)), "axes": dict(axes=[i % 3 if i < 60 else 0 for i in range(64)]),
            "empty": dict(sections=(0, 40, 24, 0))}[kind]
    axes = args.get("axes") or [a for a, s in enumerate(args["sections"]) for _ in range(s)]
    freqs = [0.9 ** f for f in range(64)]
    want = turn(x.double(), 128, pairs, freqs, axes, pos.tolist(), 1.25)
    r = Rotary(128, inv_freq=torch.tensor(freqs, dtype=torch.float64), pairs=pairs, scaling=1.25, **args)
    p = pos if wide else pos.int()
    got = rotate(x.to(DEV), r, p.to(DEV))
    check(x, got, want, 128, pairs, 1.25)
    strided = torch.stack([p, p + 1], 2).to(DEV)[:, :, 0]
    assert torch.equal(rotate(x.to(DEV), r, strided), got)
    rows = torch.cat([p, p]).to(DEV)[:n_axes]
    assert torch.equal(rotate(x.to(DEV), r, rows), got)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_places(dtype):
    """Slices of a fused projection, odd addresses, values held negated, rows in another order; results in x itself and in
    a slice of a larger tensor, whose other rows stay."""
    g = torch.Generator().manual_seed(4)
    fused = torch.randn(30, 9, 64, generator=g).to(dtype).to(DEV)
    pos = torch.arange(30, device=DEV) * 77
    r = Rotary(64, base=500.0)
    want = rotate(fused[:, 2:7].contiguous(), r, pos)
    assert torch.equal(rotate(fused[:, 2:7], r, pos), want)
    odd = torch.empty(30 * 9 * 64 + 1, dtype=dtype, device=DEV)[1:].view(30, 9, 64).copy_(fused)
    assert torch.equal(rotate(odd[:, 2:7], r, pos), want)
    assert torch.equal(rotate(fused.transpose(0, 1).contiguous().transpose(0, 1)[:, 2:7], r, pos), want)
    assert torch.equal(rotate(fused.transpose(1, 2).contiguous().transpose(1, 2)[:, 2:7], r, pos), want)
    minus = torch._neg_view(-fused)
    assert torch.equal(rotate(minus[:, 2:7], r, pos), want)
    assert torch.equal(rotate(fused[:1].expand(30, 9, 64), r, pos)[3], rotate(fused[:1], r, pos[3:4])[0])
    big = torch.full((30, 12, 64), 7.0, dtype=dtype, device=DEV)
    out = rotate(fused[:, 2:7], r, pos, out=big[:, 4:9])
    assert torch.equal(big[:, 4:9], want) and out.data_ptr() == big[:, 4:9].data_ptr()
    assert (big[:, :4] == 7).all() and (big[:, 9:] == 7).all()
    mine = fused[:, 2:7]
    assert torch.equal(rotate(mine, r, pos, out=mine), want) and torch.equal(fused[:, 2:7], want)


def test_special_values():
    """Infinities and NaN stay within their pair; large values do not pass through less than float32."""
    x = torch.ones(1, 1, 64, device=DEV).half()
    x[0, 0, 3] = float("inf")
    x[0, 0, 40] = float("nan")
    y = rotate(x, Rotary(64), torch.tensor([5], device=DEV))[0, 0]
    broken = {3, 35, 8, 40}
    assert all(bool(torch.isfinite(y[i])) != (i in broken) for i in range(64))
    z = rotate(torch.full((1, 1, 64), 65000.0, device=DEV).half(), Rotary(64), torch.tensor([0], device=DEV))
    assert (z == 65000).all()


def test_nothing_to_do():
    r = Rotary(64)
    assert rotate(torch.empty(0, 4, 64, device=DEV).half(), r, torch.empty(0, dtype=torch.int64, device=DEV)).shape == (0, 4, 64)
    assert rotate(torch.empty(3, 0, 64, device=DEV).half(), r, torch.zeros(3, dtype=torch.int64, device=DEV)).shape == (3, 0, 64)


def test_another_stream_and_a_graph():
    x = torch.randn(20, 4, 128, device=DEV).half()
    pos = torch.arange(20, device=DEV)
    r = Rotary(128)
    want = rotate(x, r, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate(x, r, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotate(x, r, pos)
    for step in range(3):
        x.copy_(torch.randn(20, 4, 128, device=DEV).half())
        pos.add_(1000 * step)
        want = rotate(x, r, pos)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_refusals():
    r = Rotary(64)
    x, pos = torch.zeros(3, 2, 64, device=DEV).half(), torch.zeros(3, dtype=torch.int64, device=DEV)
    for bad, exc in ((lambda: rotate(x.double(), r, pos), TypeError), (lambda: rotate(x[0], r, pos), TypeError),
                     (lambda: rotate(x, None, pos), TypeError), (lambda: rotate(x[..., :32], r, pos), ValueError),
                     (lambda: rotate(x, r, pos.float()), TypeError), (lambda: rotate(x, r, pos[:2]), ValueError),
                     (lambda: rotate(x, r, pos.cpu()), ValueError), (lambda: rotate(x.cpu(), r, pos), ValueError),
                     (lambda: rotate(x, r, pos[None].expand(2, 3)), ValueError),
                     (lambda: rotate(x, Rotary(64, sections=(16, 16)), pos), ValueError),
                     (lambda: rotate(x, r, pos, out=x[:2]), ValueError),
                     (lambda: rotate(x, r, pos, out=x.float()), ValueError),
                     (lambda: rotate(x, r, pos, out=x.flip(1)[:, :].transpose(0, 0)[:, [1, 0]].expand(3, 2, 64).cpu()), ValueError),
                     (lambda: rotate(x[:, :1], r, pos, out=x[:, 1:]), ValueError)):
        with pytest.raises(exc):
            bad()


def test_out_whose_rows_overlap_is_refused():
    r = Rotary(64)
    x, pos = torch.randn(3, 2, 64, device=DEV).half(), torch.arange(3, device=DEV)
    room = torch.zeros(1024, device=DEV, dtype=torch.float16)
    for strides in ((0, 64, 1), (64, 64, 1), (128, 32, 1), (127, 64, 1), (64, 191, 1)):
        with pytest.raises(ValueError):
            rotate(x, r, pos, out=room.as_strided((3, 2, 64), strides))
    assert not room.any()
    want = rotate(x, r, pos)
    for strides in ((128, 64, 1), (64, 192, 1), (300, 70, 1)):
        assert torch.equal(rotate(x, r, pos, out=room.as_strided((3, 2, 64), strides)), want)
    one = room.as_strided((1, 2, 64), (0, 64, 1))                  # a stride that nothing steps along
    assert torch.equal(rotate(x[:1], r, pos[:1], out=one), want[:1])
