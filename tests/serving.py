"""Plain forms of the serving operators for their tests: 64-bit, on the CPU, one sequence and head at
a time, with bounds for what 32-bit sums and 16-bit weights may lose."""
import math

import torch

DEV = "cuda:0"
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOOR = 2.0 ** -64


def raw(x):
    return x.view(torch.int8)


def random_cache(pages, H, bs, D, dtype, g, scale=0.02):
    """Host tensors (k, v, k_scale, v_scale) of codes spread like a model's values."""
    out = []
    for shape in ((pages, H, bs, D), (pages, H, D, bs)):
        x = torch.randn(shape, generator=g) * (QMAX[dtype] / 4)
        x = x.round().clamp(-127, 127) if dtype == torch.int8 else x.clamp(-448, 448)
        out.append(x.to(dtype))
    for _ in range(2):
        out.append((scale * (0.5 + torch.rand(pages, H, generator=g))) * (127.0 / QMAX[dtype]))
    return out


def device_cache(parts):
    from polar_pack_amd.kv_cache import KVCache
    return KVCache(*[t.to(DEV) for t in parts])


def tables(lens, bs, pages, g, width=None):
    """A block table whose rows share no page, pages in random order, -1 where none is needed."""
    need = [max(0, -(-n // bs)) for n in lens]
    width = width or max(1, max(need))
    order = torch.randperm(pages, generator=g)[:sum(need)]
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :min(n, width)] = order[at:at + min(n, width)].int()
        at += n
    return t


def offsets(news):
    return torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)


def gather(parts, table, length, h):
    """Float64 keys and values (length, D) of a sequence and head, and which tokens lie on a page."""
    k, v, ks, vs = parts
    pages, _, bs, D = k.shape
    K, V = torch.zeros(length, D, dtype=torch.float64), torch.zeros(length, D, dtype=torch.float64)
    have = torch.zeros(length, dtype=torch.bool)
    for i in range(0, length, bs):
        p = int(table[i // bs]) if i // bs < len(table) else -1
        if not 0 <= p < pages:
            continue
        n = min(bs, length - i)
        K[i:i + n] = k[p, h, :n].double() * float(ks[p, h])
        V[i:i + n] = v[p, h, :, :n].double().t() * float(vs[p, h])
        have[i:i + n] = True
    return K, V, have


def attention(q, parts, table, lens, news, causal=True, window=0, scale=None):
    """(out, lse, bound of out, bound of lse) in float64 for the rows of all sequences.

    The bounds: a score is a float32 sum of D products (D + 8 roundings of half a unit of 2^-24 of the
    sum of their magnitudes) with a few more factors, so a weight is off by a relative 2 delta; weights
    are rounded to 11 bits for the product with the values; the quotient is rounded to the output's type.
    """
    k = parts[0]
    H, bs, D = k.shape[1], k.shape[2], k.shape[3]
    n_tok, Hq = q.shape[0], q.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(n_tok, Hq, D, dtype=torch.float64)
    lse = torch.full((n_tok, Hq), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    unit = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    at = 0
    for b, n in enumerate(news):
        L = min(lens[b], table.shape[1] * bs)
        for h in range(H):
            K, V, have = gather(parts, table[b], max(L, 0), h)
            j = torch.arange(max(L, 0))
            pos = lens[b] - n + torch.arange(n)[:, None]
            seen = (j <= pos) if causal else ((j >= 0) & (pos >= 0))
            seen = seen & have
            if window:
                seen = seen & (j > pos - window)
            for hq in range(h * (Hq // H), (h + 1) * (Hq // H)):
                x = q[at:at + n, hq].double()
                s = (x @ K.t()) * scale
                s = torch.where(seen, s, -math.inf)
                any_ = seen.any(1)
                m = torch.where(any_, s.amax(1) if L > 0 else torch.zeros(n, dtype=torch.float64), 0.0)[:, None]
                w = torch.where(seen, torch.exp(s - m), 0.0)
                z = w.sum(1)
                zz = torch.where(any_, z, 1.0)
                plain = V.nan_to_num(0.0, 0.0, 0.0)          # what a row does not see does not count, NaN or not
                lost = (seen & ~V.isfinite().all(1)).any(1)
                o = torch.where(lost[:, None], math.nan, (w @ plain) / zz[:, None])
                mass = (w @ plain.abs()) / zz[:, None]
                sums = torch.where(seen, (x.abs() @ K.abs().t()) * abs(scale), 0.0)
                delta = (D + 8) * 2.0 ** -24 * (sums.amax(1) if L > 0 else torch.zeros(n, dtype=torch.float64)) + 2.0 ** -19
                out[at:at + n, hq] = torch.where(any_[:, None], o, 0.0)
                tol[at:at + n, hq] = (2 * delta[:, None] + 2.0 ** -11) * mass + unit * o.abs() + 1e-7
                lse[at:at + n, hq] = torch.where(any_, m[:, 0] + torch.log(zz), -math.inf)
                tol_lse[at:at + n, hq] = delta + 2.0 ** -16
        at += n
    return out, lse, tol, tol_lse


def append(parts, k, v, table, lens, news):
    """The cache after an append, by its float32 definition; a token at a time."""
    out = [t.clone() for t in parts]
    dtype = parts[0].dtype
    pages, H, bs, D = parts[0].shape
    at = 0
    for b, n in enumerate(news):
        first = lens[b] - n
        for blk in range(first // bs, -(-lens[b] // bs)):
            lo, hi = max(first, blk * bs), min(lens[b], blk * bs + bs)
            p = int(table[b, blk]) if 0 <= blk < table.shape[1] else -1
            if lo >= hi or not 0 <= p < pages:
                continue
            held = lo - blk * bs
            for which, new in ((0, k), (1, v)):
                x = new[at + lo - first:at + hi - first].float().transpose(0, 1)      # (H, t, D)
                c = raw(out[which])[p] if which == 0 else raw(out[which])[p].transpose(1, 2)
                sc = out[2 + which][p]
                was = sc.clone() if held else torch.zeros(H)
                need = x.abs().amax((1, 2)) / QMAX[dtype]
                now = torch.maximum(torch.maximum(was, need), torch.full((H,), FLOOR))
                top = torch.full((H,), QMAX[dtype])          # number / tensor would round the reciprocal first
                factor = torch.where(need == now, top / x.abs().amax((1, 2)), torch.ones(H) / now)
                for h in range(H):
                    ok = bool(torch.isfinite(now[h]))
                    if held and (not ok or now[h] > was[h]):
                        old = c[h, :held].clone().view(dtype).float() * (was[h] / now[h])
                        c[h, :held] = raw(round_codes(old, dtype)) if ok else 0
                    c[h, held:held + hi - lo] = raw(round_codes(x[h] * factor[h], dtype)) if ok else 0
                sc.copy_(now)
        at += n
    return out


def round_codes(x, dtype):
    q = QMAX[dtype]
    return (x.round() if dtype == torch.int8 else x).clamp(-q, q).to(dtype)
