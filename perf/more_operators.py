"""More serving operators around the packed Linears: rotary positions, the cache's append with the
rotation on the way, a 4-bit key/value cache with its attention, and the check of drafted tokens.

The 4-bit cache holds codes e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the
earlier one in the low half: K (pages, heads, block, D / 2) and V (pages, heads, D, block / 2).  Every 32
values of a token and head share a scale, a power of two held as float8 e5m2: K (pages, heads,
block, D / 32), V (pages, heads, D / 32, block).  The 8-bit cache is that of ``perf/operators.py``.  Queries, keys and
values are slices of one fused projection's output.  The 3B-shaped model of the package's benchmark has 16 query
heads and 2 key/value heads of 128 and a vocabulary of 151,936; its four packed models decode in lock step.
"""
import math

import torch

own = False
DEV = "cuda:0"
FLOOR = 2.0 ** -64                     # smallest scale of a page of the 8-bit cache
QMAX = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
VOCAB = 151936
BASE = 1000000.0                       # of the angles' frequencies


def listed():
    return [
        # one decode step of the four packed models: each one's queries and keys
        {"name": "rotate_step", "op": "rotate", "T": 4, "heads": 18, "D": 128, "rot": 128, "pairs": "halves", "axes": 1,
         "type": "f16"},
        # a batch of pictures and films: time, height and width turn their own frequencies
        {"name": "rotate_video", "op": "rotate", "T": 16200, "heads": 18, "D": 128, "rot": 128, "pairs": "halves",
         "axes": 3, "type": "bf16"},
        # that decode step as a layer runs it: queries and keys turned, keys and values appended
        {"name": "append_step", "op": "append", "B": 4, "lo": 901, "hi": 1130, "new": 1, "Hq": 16, "H": 2, "D": 128,
         "rot": 128, "pairs": "halves", "axes": 1, "block": 64, "codes": "int8", "type": "f16"},
        # the four models take in a prompt with a picture
        {"name": "append_prompt", "op": "append", "B": 4, "lo": 2048, "hi": 2048, "new": 2048, "Hq": 16, "H": 2,
         "D": 128, "rot": 128, "pairs": "halves", "axes": 3, "block": 64, "codes": "int8", "type": "f16"},
        # a serving batch's decode step into the 4-bit cache
        {"name": "append4_batch", "op": "append", "B": 64, "lo": 77, "hi": 8190, "new": 1, "Hq": 32, "H": 8, "D": 128,
         "rot": 64, "pairs": "neighbours", "axes": 1, "block": 64, "codes": "e2m1", "type": "bf16"},
        # ragged prompts behind cached prefixes into the 4-bit cache, many heads
        {"name": "append4_ragged", "op": "append", "B": 16, "lo": 1203, "hi": 4999, "new": 1200, "Hq": 32, "H": 8,
         "D": 128, "rot": 128, "pairs": "halves", "axes": 1, "block": 32, "codes": "e2m1", "type": "bf16"},
        # attention of the four models' decode step to the 4-bit cache
        {"name": "attend4_step", "op": "attend", "B": 4, "lo": 901, "hi": 1130, "new": 1, "Hq": 16, "H": 2, "D": 128,
         "block": 64, "type": "f16", "window": 0},
        # a serving batch of unequal lengths
        {"name": "attend4_batch", "op": "attend", "B": 64, "lo": 77, "hi": 8190, "new": 1, "Hq": 32, "H": 8, "D": 128,
         "block": 64, "type": "bf16", "window": 0},
        # few sequences, long contexts: what a cache of 4 bits is for
        {"name": "attend4_long", "op": "attend", "B": 4, "lo": 200003, "hi": 262144, "new": 1, "Hq": 16, "H": 2,
         "D": 128, "block": 64, "type": "f16", "window": 0},
        # a piece of one long prompt, taken in by pieces
        {"name": "attend4_piece", "op": "attend", "B": 1, "lo": 32701, "hi": 32701, "new": 509, "Hq": 16, "H": 2,
         "D": 128, "block": 64, "type": "bf16", "window": 0},
        # the four models check four drafted tokens each
        {"name": "verify_step", "op": "verify", "B": 4, "n": 4, "V": VOCAB, "type": "f32", "draft": True, "ragged": False},
        # a serving batch that drafts five tokens a sequence, some fewer
        {"name": "verify_batch", "op": "verify", "B": 128, "n": 5, "V": VOCAB, "type": "f32", "draft": True,
         "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotate", "append", "append", "attend", "attend", "verify"))
    if op == "verify":
        while True:
            B, n, V = _log_int(rng, 1, 256), rng.randint(1, 8), _log_int(rng, 1000, VOCAB)
            if B * (n + 1) * V <= 128 * 6 * VOCAB:
                break
        return {"op": op, "B": B, "n": n, "V": V, "type": rng.choice(("f32", "f32", "bf16", "f16")),
                "draft": rng.random() < 0.75, "ragged": rng.random() < 0.5}
    if op == "rotate":
        D = rng.choice((64, 80, 96, 128, 192, 256))
        while True:
            T, heads = _log_int(rng, 1, 20000), _log_int(rng, 1, 40)
            if T * heads * D <= 16200 * 18 * 128:
                break
        return {"op": op, "T": T, "heads": heads, "D": D, "rot": rng.choice((D, D, D // 32 * 16)),
                "pairs": rng.choice(("halves", "neighbours")), "axes": rng.choice((1, 3)),
                "type": rng.choice(("f16", "bf16", "f32"))}
    Hq, H, D = rng.choice(((16, 2, 128), (32, 8, 128), (32, 8, 64), (8, 8, 128), (16, 1, 256), (12, 4, 192)))
    while True:
        B, hi = _log_int(rng, 1, 64), _log_int(rng, 16, 40000)
        new = 1 if op == "attend" and rng.random() < 0.5 else _log_int(rng, 1, 2048)
        new = min(new, hi)
        lo = max(new, int(hi * rng.uniform(0.1, 1.0)))
        if B * hi * H * D <= 1 << 28 and B * new * hi * Hq * D <= 1 << 34 and B * new * Hq * D <= 1 << 26:
            break
    case = {"op": op, "B": B, "lo": lo, "hi": hi, "new": new, "Hq": Hq, "H": H, "D": D,
            "block": rng.choice((16, 32, 64, 128)), "type": rng.choice(("f16", "bf16"))}
    if op == "attend":
        case["window"] = rng.choice((0, 0, max(1, hi // 3)))
    else:
        case |= {"codes": rng.choice(("int8", "e4m3", "e2m1", "e2m1")), "rot": rng.choice((D, D, D // 2)),
                 "pairs": rng.choice(("halves", "neighbours")), "axes": rng.choice((1, 3))}
    return case


def _lengths(case):
    """Tokens of each sequence after the call: spread over [lo, hi], the last one hi."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [int(lo + (hi - lo) * ((i + 1) * 0.6180339887 % 1.0)) for i in range(B - 1)] + [hi]


def _news(case):
    """New tokens of each sequence: `new`, or fewer for some sequences of a batch of prompts."""
    B, new = case["B"], case["new"]
    return [new if new < 16 or case["lo"] == case["hi"] else max(1, new - (37 * i) % (new // 2)) for i in range(B)]


def _drafts(case):
    """Drafted tokens of each sequence."""
    return [case["n"] - (b % 3 if case["ragged"] and case["n"] > 2 else 0) for b in range(case["B"])]


def _back(case):
    """Tokens of each sequence that an append is read back by: the new ones, and where they share a page's scale with
    earlier ones those too."""
    lens, news, bs = _lengths(case), _news(case), case["block"]
    return news if case["codes"] == "e2m1" else [L - (L - n) // bs * bs for L, n in zip(lens, news)]


def _sections(case):
    """How many frequencies each axis turns: of three a quarter the first, the rest halved, in runs of 8."""
    f = case["rot"] // 2
    return [f] if case["axes"] == 1 else [f - 2 * (f * 3 // 64 * 8), f * 3 // 64 * 8, f * 3 // 64 * 8]


def work(case):
    es = torch.empty((), dtype=TYPES[case["type"]]).element_size()
    if case["op"] == "rotate":
        n = case["T"] * case["heads"] * case["D"]
        return {"bytes": 2 * n * es + 8 * case["T"] * case["axes"], "flops": 3 * case["T"] * case["heads"] * case["rot"]}
    if case["op"] == "verify":
        # every sequence's row of the target, and one of the draft where a token is refused: about half of them
        rows = case["B"] * (1.5 if case["draft"] else 1.0)
        return {"bytes": int(rows * case["V"] * es), "flops": int(3 * rows * case["V"])}
    H, Hq, D, bs = case["H"], case["Hq"], case["D"], case["block"]
    lens, news = _lengths(case), _news(case)
    if case["op"] == "append":
        n, back = sum(news), sum(_back(case))
        bits = 4.25 if case["codes"] == "e2m1" else 8
        # queries read and written, new values read, codes written; then codes read and their values written
        return {"bytes": int(2 * n * Hq * D * es + 2 * H * D * (n * (es + bits / 8) + back * (bits / 8 + es))),
                "flops": 3 * n * (Hq + H) * case["rot"] + 2 * H * D * (6 * n + 2 * back)}
    w = case["window"]
    pairs, seen = 0, 0
    for L, n in zip(lens, news):
        first = L - n
        if w:
            pairs += sum(min(p + 1, w) for p in range(first, L))
            seen += min(L, w + n - 1)
        else:
            pairs += n * first + n * (n + 1) // 2
            seen += L
    return {"bytes": int(2 * seen * H * D * 4.25 / 8) + 2 * sum(news) * Hq * D * es, "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------------------------ inputs

def _grid(T, g):
    """Positions (3, T) of texts and pictures one after another: text steps all axes, a picture's rows and columns
    their own."""
    i = torch.arange(T, device=DEV)
    part, at = i // 700, i % 700                       # 100 words, then a picture of 20 rows of 30
    first = part * 130
    spot = (at - 100).clamp(min=0)
    word = at < 100
    pos = [torch.where(word, first + at, first + 100 + e) for e in (0 * i, spot // 30, spot % 30)]
    return torch.stack(pos) + int(torch.randint(0, 50, (1,), generator=g, device=DEV))


def _angles(case, s, T, g):
    """What a rotation knows: frequencies, whose axis each is, positions (None: the tokens' own)."""
    f = case["rot"] // 2
    s["inv_freq"] = BASE ** (-torch.arange(f, dtype=torch.float64, device=DEV) / f)
    s["axis"] = torch.repeat_interleave(torch.arange(case["axes"], device=DEV),
                                        torch.tensor(_sections(case), device=DEV))
    s["positions"] = _grid(T, g) if case["axes"] == 3 else None


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]
    s = {"op": case["op"], "case": case}
    if case["op"] == "rotate":
        T, heads, D = case["T"], case["heads"], case["D"]
        spread = torch.exp(0.5 * torch.randn(heads, D, generator=g, device=DEV))
        # queries and keys, the first `heads` heads of a fused projection's output
        fused = torch.randn(T, heads + 2, D, generator=g, device=DEV)
        fused[:, :heads].mul_(spread)
        s["x"] = fused.to(dt)[:, :heads]
        _angles(case, s, T, g)
        if s["positions"] is None:                     # a batch of tokens of texts of any length
            s["positions"] = torch.randint(0, 131072, (T,), generator=g, device=DEV)
        return s
    if case["op"] == "verify":
        B, n, V = case["B"], case["n"], case["V"]
        s["p"] = torch.empty(B, n + 1, V, dtype=dt, device=DEV)
        s["q"] = torch.empty(B, n, V, dtype=dt, device=DEV) if case["draft"] else None
        s["tokens"] = torch.empty(B, n, dtype=torch.int64, device=DEV)
        for b in range(B):
            # a few words far above a broad bell; the draft knows the bell well and the words roughly
            x = torch.randn(n + 1, V, generator=g, device=DEV).mul_(2.0)
            words = torch.randint(0, V, (n + 1, 4), generator=g, device=DEV)
            x.scatter_(1, words, 9 + 5 * torch.rand(n + 1, 4, generator=g, device=DEV))
            s["p"][b] = torch.softmax(x, 1).to(dt)
            y = x[:n] + 0.4 * torch.randn(n, V, generator=g, device=DEV)
            d = torch.softmax(y, 1)
            s["tokens"][b] = torch.multinomial(d, 1, generator=g)[:, 0]
            if s["q"] is not None:
                s["q"][b] = d.to(dt)
        s["uniforms"] = torch.rand(B, n + 1, generator=g, device=DEV)
        s["counts"] = torch.tensor(_drafts(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
        return s
    B, H, Hq, D, bs = case["B"], case["H"], case["Hq"], case["D"], case["block"]
    kind = case.get("codes", "e2m1")
    lens, news = _lengths(case), _news(case)
    width = max(-(-L // bs) for L in lens)
    pages = B * width + 3
    order = torch.randperm(pages, generator=g, device=DEV)[:B * width].int()
    s |= {"table": order.view(B, width).contiguous(), "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
          "cu": None, "D": D, "bs": bs, "H": H, "G": Hq // H}
    if case["new"] > 1:
        s["cu"] = torch.tensor([sum(news[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV)
    # keys have channels of unequal size
    spread = torch.exp(0.5 * torch.randn(Hq + 2 * H, D, generator=g, device=DEV))
    qkv = torch.randn(sum(news), Hq + 2 * H, D, generator=g, device=DEV).mul_(spread).to(dt)
    s["qnew"], s["knew"], s["vnew"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    if case["op"] == "append":
        back = _back(case)
        s["cu_read"] = torch.tensor([sum(back[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV)
        s["total"] = sum(back)
        _angles(case, s, sum(news), g)
    if kind == "e2m1":
        # codes as a bell leaves them, by 256 equally likely quantiles; scales within a factor of four
        bell = torch.special.ndtri((torch.arange(256, device=DEV) + 0.5) / 256) * 2.5
        nibble = _e2m1(bell).to(torch.uint8)
        for n, shape, sshape in (("k", (pages, H, bs, D // 2), (pages, H, bs, D // 32)),
                                 ("v", (pages, H, D, bs // 2), (pages, H, D // 32, bs))):
            codes = torch.empty(shape, dtype=torch.uint8, device=DEV)
            for p in range(0, pages, 4096):
                at = [torch.randint(0, 256, codes[p:p + 4096].shape, generator=g, device=DEV, dtype=torch.uint8)
                      for _ in range(2)]
                codes[p:p + 4096] = nibble[at[0].int()] | nibble[at[1].int()] << 4
            s[n] = codes
            e = torch.randint(-3, 0, sshape, generator=g, device=DEV, dtype=torch.int8)
            s[n + "s"] = torch.exp2(e.to(torch.float32)).to(torch.float8_e5m2)
        return s
    for n, shape in (("k", (pages, H, bs, D)), ("v", (pages, H, D, bs))):
        codes = torch.empty(shape, dtype=torch.int8, device=DEV)
        for p in range(0, pages, 4096):
            part = torch.randn(codes[p:p + 4096].shape, generator=g, device=DEV)
            if kind == "int8":
                codes[p:p + 4096] = part.mul_(30).round_().clamp_(-127, 127).to(torch.int8)
            else:
                codes[p:p + 4096] = part.mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)
        s[n] = codes.view(CODES[kind])
        s[n + "s"] = (0.02 + 0.02 * torch.rand(pages, H, generator=g, device=DEV)) * (127 / QMAX[kind])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from polar_pack_amd.kv_cache import KVCache, KVCache4
        from polar_pack_amd.rotary import Rotary
        if "k" in s:
            s["cache"] = (KVCache4 if case.get("codes", "e2m1") == "e2m1" else KVCache)(s["k"], s["v"], s["ks"], s["vs"])
        if "inv_freq" in s:
            s["rotary"] = Rotary(case["D"], rotary_dim=case["rot"], base=BASE, pairs=case["pairs"],
                                 sections=_sections(case), device=DEV)
    return s


# --------------------------------------------------------------------------- plain forms

def _tokens(s):
    """(sequence, position, page, place in the page) of every new token, and their first positions."""
    cu, lens, B = s["cu"], s["lens"].long(), s["table"].shape[0]
    if cu is None:
        seq, nth, n = torch.arange(B, device=DEV), torch.zeros(B, dtype=torch.long, device=DEV), 1
    else:
        at = torch.arange(s["qnew"].shape[0], device=DEV)
        seq = torch.bucketize(at, cu[1:].long(), right=True)
        nth, n = at - cu.long()[seq], (cu[1:] - cu[:-1]).long()
    first = lens - n
    pos = first[seq] + nth
    return seq, pos, s["table"][seq, pos // s["bs"]].long(), pos % s["bs"], first


def _turn(s, x, positions, dtype):
    """x (T, heads, D) turned, computed and left in `dtype`; angles in 64 bits, which far positions need."""
    case, rot = s["case"], s["case"]["rot"]
    pos = positions if positions.dim() == 2 else positions[None]
    angle = pos.double()[s["axis"]].t() * s["inv_freq"]                     # (T, rot / 2)
    c, sn = torch.cos(angle).to(dtype)[:, None], torch.sin(angle).to(dtype)[:, None]
    x = x.to(dtype)
    out = x.clone()
    a, b = ((x[..., :rot // 2], x[..., rot // 2:rot]) if case["pairs"] == "halves"
            else (x[..., :rot:2], x[..., 1:rot:2]))
    first, second = a * c - b * sn, b * c + a * sn
    if case["pairs"] == "halves":
        out[..., :rot // 2], out[..., rot // 2:rot] = first, second
    else:
        out[..., :rot:2], out[..., 1:rot:2] = first, second
    return out


def _round_codes(x, codes):
    if codes == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _raw(x):
    """Codes as bytes: float8 tensors take no indexed writes."""
    return x.view(torch.int8)


def _e2m1(t):
    """The code (0..15, sign in bit 3) nearest to each number, halfway ones to the even code."""
    a = t.abs()
    n = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    return n + 8 * (t < 0)


def _values4(codes):
    """Bytes (..., n) as the numbers (..., 2 n) of their codes."""
    lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=DEV)
    return torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], -1).flatten(-2)


def _group(x):
    """(nibbles, scales) of rows (..., D) in groups of 32: the smallest power of two from 2^-14 to 2^13 that is a
    seventh of the largest or more."""
    v = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(v.abs().amax(-1))                                    # m in [0.5, 1)
    e = (e - 3 + (m > 0.875)).clamp(-14, 13)
    e = torch.where(m == 0, -14, e).to(x.dtype)
    return _e2m1((v * torch.exp2(-e)[..., None]).clamp(-6, 6)).flatten(-2), torch.exp2(e)


def _plain_append4(s, k, page, place):
    for name, x in (("k", k), ("v", s["vnew"].float())):
        nib, scale = _group(x)
        nib, codes = nib.to(torch.uint8), s[name]
        byte = scale.to(torch.float8_e5m2).view(torch.int8)
        if name == "k":
            codes[page, :, place] = nib[..., 0::2] | nib[..., 1::2] << 4
            _raw(s["ks"])[page, :, place] = byte
        else:
            for odd in (0, 1):                                              # two tokens share a byte
                at = place % 2 == odd
                p, t = page[at], place[at] // 2
                codes[p, :, :, t] = codes[p, :, :, t] & (15 if odd else 240) | nib[at] << 4 * odd
            _raw(s["vs"])[page, :, :, place] = byte


def _plain_append8(s, knew, seq, page, place, first):
    kind, qmax = s["case"]["codes"], QMAX[s["case"]["codes"]]
    old = first % s["bs"]                              # tokens before the new ones in a sequence's first page
    head = s["table"][torch.arange(len(old), device=DEV), torch.div(first, s["bs"], rounding_mode="floor")].long()
    kept = torch.arange(s["bs"], device=DEV) < old[:, None]
    for name, x in (("k", knew), ("v", s["vnew"].float())):
        codes, scale = s[name], s[name + "s"]
        before = torch.zeros_like(scale)
        before[head] = torch.where(old[:, None] > 0, scale[head], 0.0)
        top = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(-1, s["H"]), x.abs().amax(-1), "amax")
        now = torch.maximum(torch.maximum(before, top / qmax), torch.full_like(top, FLOOR))
        ratio = before[head] / now[head]
        prev = codes[head].float()
        mask = kept[:, None, :, None] if name == "k" else kept[:, None, None, :]
        grown = mask & (now[head] > before[head])[:, :, None, None]
        part = torch.where(grown, _raw(_round_codes(prev * ratio[:, :, None, None], kind)), _raw(codes)[head])
        _raw(codes)[head] = part
        scale[page] = now[page]
        c = _raw(_round_codes(x * (1.0 / now[page])[:, :, None], kind))
        if name == "k":
            _raw(codes)[page, :, place] = c
        else:
            _raw(codes)[page, :, :, place] = c


def _plain_append(s):
    seq, pos, page, place, first = _tokens(s)
    at = pos if s["positions"] is None else s["positions"]
    if s["case"]["codes"] == "e2m1":
        # in 64 bits: a step of 4 bits is wide, and next to a border a small error is one of a step
        _plain_append4(s, _turn(s, s["knew"], at, torch.float64), page, place)
    else:
        _plain_append8(s, _turn(s, s["knew"], at, torch.float32), seq, page, place, first)
    return _turn(s, s["qnew"], at, torch.float32).to(s["qnew"].dtype)


def _plain_read(s, dt):
    """Values of each sequence's last cu_read[b + 1] - cu_read[b] tokens, one sequence after another."""
    cu, lens, H, D = s["cu_read"].long(), s["lens"].long(), s["H"], s["D"]
    at = torch.arange(s["total"], device=DEV)
    seq = torch.bucketize(at, cu[1:], right=True)
    pos = lens[seq] - cu[seq + 1] + at
    page, place = s["table"][seq, pos // s["bs"]].long(), pos % s["bs"]
    if s["case"]["codes"] == "e2m1":
        k = _values4(s["k"][page, :, place])
        odd = (place % 2)[:, None, None]
        v = s["v"][page, :, :, place // 2]
        v = _values4(torch.where(odd == 1, v >> 4, v & 15)[..., None])[..., 0]
        ks = _raw(s["ks"])[page, :, place].view(torch.float8_e5m2).float()
        vs = _raw(s["vs"])[page, :, :, place].view(torch.float8_e5m2).float()
        return [(x.unflatten(-1, (-1, 32)) * y[..., None]).flatten(-2).to(dt) for x, y in ((k, ks), (v, vs))]
    k = _raw(s["k"])[page, :, place].view(s["k"].dtype).float() * s["ks"][page][:, :, None]
    v = _raw(s["v"])[page, :, :, place].view(s["v"].dtype).float() * s["vs"][page][:, :, None]
    return [k.to(dt), v.to(dt)]


def _plain_attend(s):
    B, H, G, D, bs = s["table"].shape[0], s["H"], s["G"], s["D"], s["bs"]
    case = s["case"]
    n, width = max(_news(case)), s["table"].shape[1]
    seq, pos, _, _, first = _tokens(s)
    nth = pos - first[seq]
    q = torch.zeros(B, n, H, G, D, device=DEV)
    q[seq, nth] = s["qnew"].float().reshape(-1, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    table = s["table"].long()
    # (B, width, H, block, D)
    k = _values4(s["k"][table]).unflatten(-1, (-1, 32)).mul_(_raw(s["ks"])[table].view(torch.float8_e5m2).float()[..., None])
    kt = k.flatten(-2).permute(0, 2, 4, 1, 3).reshape(B, H, D, width * bs).contiguous()
    del k
    sc = torch.matmul(q, kt) * (1.0 / math.sqrt(D))
    del kt
    key = torch.arange(width * bs, device=DEV)
    at = (first[:, None] + torch.arange(n, device=DEV))[:, :, None]
    seen = key <= at
    if case["window"]:
        seen &= key > at - case["window"]
    sc = sc.view(B, H, G, n, width * bs).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, H, G * n, width * bs)
    del sc
    # (B, width, H, D, block)
    v = _values4(s["v"][table]).unflatten(3, (-1, 32)).mul_(_raw(s["vs"])[table].view(torch.float8_e5m2).float()[:, :, :, :, None])
    v = v.flatten(3, 4).permute(0, 2, 1, 4, 3).reshape(B, H, width * bs, D).contiguous()
    o = torch.matmul(p, v).view(B, H, G, n, D).permute(0, 3, 1, 2, 4)
    return o[seq, nth].reshape(-1, H * G, D).to(s["qnew"].dtype)


def _plain_verify(s):
    p, q, tokens, u = s["p"], s["q"], s["tokens"], s["uniforms"].double()
    B, n, V = p.shape[0], p.shape[1] - 1, p.shape[2]
    b = torch.arange(B, device=DEV)
    count = torch.full((B,), n, device=DEV) if s["counts"] is None else s["counts"].long()
    pd = p[:, :n].gather(2, tokens[..., None])[..., 0].double()
    qd = 1.0 if q is None else q.gather(2, tokens[..., None])[..., 0].double()
    good = (u[:, :n] * qd < pd) & (torch.arange(n, device=DEV) < count[:, None])
    accepted = good.long().cumprod(1).sum(1)
    at = accepted.clamp(max=n - 1)
    refused = accepted < count
    # in 64 bits: what decides is where a long sum passes a number
    row = p[b, accepted].double()
    if q is None:
        less = torch.zeros_like(row).scatter_(1, tokens[b, at][:, None], row.gather(1, tokens[b, at][:, None]))
    else:
        less = q[b, at].double()
    rest = torch.where(refused[:, None], (row - less).clamp(min=0), row)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, row)
    sums = rest.cumsum(1)
    pick = (sums > (u[b, n] * sums[:, -1])[:, None]).long().argmax(1)
    out = torch.where(torch.arange(n + 1, device=DEV) < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    return [out.scatter(1, accepted[:, None], pick[:, None]), accepted]


def run(s):
    """One pass: rotate, append (and what was written read back), attend, or check drafted tokens."""
    if own:
        from polar_pack_amd import drafts, kv_cache, rotary
        if s["op"] == "rotate":
            return rotary.rotate(s["x"], s["rotary"], s["positions"])
        if s["op"] == "verify":
            r = drafts.verify_drafts(s["p"], s["q"], s["tokens"], s["uniforms"], s["counts"])
            return [r.tokens, r.accepted]
        c = s["cache"]
        if s["op"] == "attend":
            return kv_cache.kv_attention(s["qnew"], c, s["table"], s["lens"], s["cu"], window=s["case"]["window"])
        q = kv_cache.kv_rotate_append(c, s["qnew"], s["knew"], s["vnew"], s["rotary"], s["table"], s["lens"], s["cu"],
                                      positions=s["positions"])
        k, v = kv_cache.kv_read(c, s["table"], s["lens"], s["cu_read"], total=s["total"], dtype=s["knew"].dtype)
        return [q, k, v] + ([] if s["case"]["codes"] == "e2m1" else [c.k_scale, c.v_scale])
    if s["op"] == "rotate":
        return _turn(s, s["x"], s["positions"], torch.float32).to(s["x"].dtype)
    if s["op"] == "verify":
        return _plain_verify(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    q = _plain_append(s)
    return [q, *_plain_read(s, s["knew"].dtype)] + ([] if s["case"]["codes"] == "e2m1" else [s["ks"], s["vs"]])


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_turn(case, s, x, positions):
    """Pairs as complex numbers, turned by e^(i angle)."""
    rot = case["rot"]
    axis = [a for a, n in enumerate(_sections(case)) for _ in range(n)]
    freq = torch.tensor([BASE ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=DEV)
    at = torch.stack([positions[a] if positions.dim() == 2 else positions for a in axis], 1).double()
    turn = torch.polar(torch.ones_like(at * freq), at * freq)[:, None]
    y = x.double()
    if case["pairs"] == "halves":
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * turn
        return torch.cat([z.real, z.imag, y[..., rot:]], -1)
    z = torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), y[..., rot:]], -1)


def _nearest4(x):
    """Values of the 4-bit cache nearest to x (..., D)."""
    v = x.unflatten(-1, (-1, 32))
    scale = torch.full_like(v[..., :1], 2.0 ** -14)
    for e in range(-13, 14):
        scale = torch.where(v.abs().amax(-1, keepdim=True) > 7 * 2.0 ** (e - 1), 2.0 ** e, scale)
    code = torch.zeros_like(v)
    for lo, hi, up in zip(E2M1, E2M1[1:], (False, True) * 4):               # halfway: up to even codes, every second one
        mid = (lo + hi) / 2
        over = v.abs() / scale
        code = torch.where((over >= mid) if up else (over > mid), hi, code)
    return (torch.copysign(code, v) * scale).flatten(-2)


def _exact_append(case, s):
    kind, bs = case["codes"], case["block"]
    lens, news = _lengths(case), _news(case)
    own_places = torch.cat([torch.arange(L - n, L, device=DEV) for L, n in zip(lens, news)])
    at = own_places if s["positions"] is None else s["positions"]
    q, knew = _exact_turn(case, s, s["qnew"], at), _exact_turn(case, s, s["knew"], at)
    if kind == "e2m1":
        return [q, _nearest4(knew), _nearest4(s["vnew"].double())]
    table = s["table"].cpu().tolist()
    qmax, new_values = QMAX[kind], {"k": knew, "v": s["vnew"].double()}
    outs, scales, at = {"k": [], "v": []}, {}, 0
    rounded = (lambda x: x.round().clamp(-127, 127)) if kind == "int8" else \
        (lambda x: x.clamp(-448, 448).to(torch.float8_e4m3fn).double())
    for name in "kv":
        scales[name] = s[name + "s"].double()
    for b, (L, n) in enumerate(zip(lens, news)):
        first = L - n
        for blk in range(first // bs, -(-L // bs)):
            page, lo, hi = table[b][blk], max(first, blk * bs), min(L, blk * bs + bs)
            held = lo - blk * bs
            for name in "kv":
                x = new_values[name][at + lo - first:at + hi - first]                  # (t, H, D)
                c = s[name][page].double()
                c = c if name == "k" else c.transpose(1, 2)                            # (H, bs, D)
                was = scales[name][page].clone() if held else torch.zeros_like(scales[name][page])
                now = torch.maximum(was, x.abs().amax((0, 2)) / qmax).clamp(min=FLOOR)
                prev = c[:, :held] * (was / now)[:, None, None]
                prev = torch.where((now > was)[:, None, None], rounded(prev), c[:, :held])
                new = rounded(x.transpose(0, 1) / now[:, None, None])
                outs[name].append((torch.cat([prev, new], 1) * now[:, None, None]).transpose(0, 1))
                scales[name][page] = now
        at += n
    return [q, torch.cat(outs["k"]), torch.cat(outs["v"]), scales["k"], scales["v"]]


def _exact_attend(case, s):
    H, G, D, bs, w = case["H"], case["Hq"] // case["H"], case["D"], case["block"], case["window"]
    number = torch.tensor([(-1) ** (c >> 3) * E2M1[c & 7] for c in range(16)], dtype=torch.float64, device=DEV)
    out, at = torch.empty(s["qnew"].shape, dtype=torch.float64, device=DEV), 0
    for b, (L, n) in enumerate(zip(_lengths(case), _news(case))):
        pages = s["table"][b, :-(-L // bs)].long()
        where = torch.arange(L - n, L, device=DEV)[:, None]
        key = torch.arange(L, device=DEV)
        hidden = key > where
        if w:
            hidden |= key <= where - w
        for h in range(H):
            kc, vc = s["k"][:, h][pages].int(), s["v"][:, h][pages].int()
            kd, vd = (torch.stack([number[c % 16], number[c // 16]], -1).flatten(-2) for c in (kc, vc))
            ks = s["ks"].view(torch.uint8)[:, h][pages].view(torch.float8_e5m2).double().repeat_interleave(32, 2)
            vs = s["vs"].view(torch.uint8)[:, h][pages].view(torch.float8_e5m2).double().repeat_interleave(32, 1)
            kd = (kd * ks).reshape(-1, D)[:L].t().contiguous()
            vd = (vd * vs).transpose(1, 2).reshape(-1, D)[:L].contiguous()
            for j in range(h * G, h * G + G):
                logit = (s["qnew"][at:at + n, j].double() @ kd) / math.sqrt(D)
                out[at:at + n, j] = torch.softmax(logit.masked_fill(hidden, -math.inf), 1) @ vd
        at += n
    return out


def _exact_verify(case, s):
    n, tokens, accepted = case["n"], [], []
    u, d = s["uniforms"].double().tolist(), s["tokens"].tolist()
    for b, count in enumerate(_drafts(case)):
        k = 0
        while k < count:
            qd = 1.0 if s["q"] is None else float(s["q"][b, k, d[b][k]])
            if not u[b][k] * qd < float(s["p"][b, k, d[b][k]]):
                break
            k += 1
        rest = s["p"][b, k].double()
        if k < count:
            other = rest.clone()
            if s["q"] is None:
                other[d[b][k]] = 0
            else:
                other = (rest - s["q"][b, k].double()).clamp(min=0)
            rest = other if float(other.sum()) > 0 else rest
        sums = rest.cumsum(0)
        tokens.append(d[b][:k] + [int(torch.searchsorted(sums, u[b][n] * sums[-1], right=True))] + [-1] * (n - k))
        accepted.append(k)
    return [torch.tensor(tokens, device=DEV), torch.tensor(accepted, device=DEV)]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotate":
        return _exact_turn(case, s, s["x"], s["positions"])
    return {"append": _exact_append, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](case, s)
