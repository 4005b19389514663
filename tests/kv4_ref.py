"""The paged 4-bit cache, its norms and its attention in 64 bits, from the description of a page."""

import math

import torch

MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pow2(e):
    """2^e of whole e from -400 to 400, exactly (the device's pow is not)."""
    return torch.tensor([2.0 ** i for i in range(-400, 401)], dtype=torch.float64, device=e.device)[e.long() + 400]


def quantize(x):
    """(codes as one number an element, scale bytes) of x (..., hd): every magnitude looked at, ties to the even code."""
    x = x.double().unflatten(-1, (x.shape[-1] // 32, 32))
    top = x.abs().amax(-1)
    finite = x.isfinite().all(-1)
    t = torch.where(finite, top, torch.zeros_like(top))
    e = torch.frexp(t)[1].double() - 4         # t >= 2^(e + 3): the least e is e, e + 1 or (beyond 7 / 8) e + 2
    for _ in range(2):
        e = torch.where(t > 7 * pow2(e.clamp(-300, 300)), e + 1, e)
    e = torch.where(t > 0, e, torch.full_like(e, -100.0)).clamp(-100, 125)
    y = torch.where(finite[..., None], x, torch.zeros_like(x)) * pow2(-e)[..., None]
    code, dist = torch.zeros_like(y), torch.full_like(y, math.inf)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):
        d = (y.abs() - MAGS[c]).abs()
        code, dist = torch.where(d < dist, torch.full_like(y, float(c)), code), torch.minimum(d, dist)
    code = code.long() + 8 * (y < 0).long()
    return code.flatten(-2), torch.where(finite, e.long() + 127, torch.full_like(e, 255).long())


def value(code, scale):
    """Elements (..., hd) of codes and scale bytes (..., hd / 32)."""
    m = torch.tensor(MAGS + tuple(-v for v in MAGS), dtype=torch.float64, device=code.device)[code.long()]
    f = pow2(scale.long() - 127)
    f = torch.where(scale == 255, torch.full_like(f, math.nan), f)
    return (m.unflatten(-1, (scale.shape[-1], 32)) * f[..., None]).flatten(-2)


def places(hd, device="cpu"):
    """Byte offsets in a tile: (token, element) -> key code, value code; (token, block) -> key scale, value scale."""
    t = torch.arange(16, device=device)[:, None]
    c, b, run = torch.arange(hd, device=device), torch.arange(hd // 32, device=device), hd // 16
    return (t * (hd // 2) + c // 2, 8 * hd + t // 4 * (2 * hd) + c // run * (2 * run) + t % 4 * (run // 2) + c % run // 2,
            16 * hd + t * (hd // 32) + b, 16 * hd + hd // 2 + (t // 4 * (hd // 32) + b) * 4 + t % 4)


def rows_of(pages, table_row):
    """A sequence's keys and values (n_kv, slots, hd) in 64 bits; where there is no page NaN."""
    hd = pages.shape[3] // 17
    pk, pv, sk, sv = places(hd, pages.device)
    there = (table_row >= 0) & (table_row < pages.shape[0])
    raw = pages[torch.where(there, table_row, torch.zeros_like(table_row)).long()].permute(1, 0, 2, 3).flatten(1, 2)
    shift = (torch.arange(hd, device=pages.device) % 2) * 4
    out = []
    for codes, scales in ((pk, sk), (pv, sv)):
        x = value(((raw[:, :, codes].int() >> shift) & 15), raw[:, :, scales]).flatten(1, 2)
        gone = ~there.repeat_interleave(pages.shape[2] * 16)
        out.append(x.masked_fill(gone[None, :, None], math.nan))
    return out


def store(pages, table, b, slot, k, v):
    """k, v (n_kv, hd) into slot ``slot`` of sequence b, byte by byte."""
    hd, tiles = pages.shape[3] // 17, pages.shape[2]
    pk, pv, sk, sv = places(hd)
    page, off = int(table[b, slot // (16 * tiles)]), slot % (16 * tiles)
    tok = off % 16
    for x, codes, scales in ((k, pk, sk), (v, pv, sv)):
        c, s = quantize(x)
        tile = pages[page, :, off // 16]
        tile[:, codes[tok][0::2].to(tile.device)] = (c[:, 0::2] | c[:, 1::2] << 4).to(torch.uint8)
        tile[:, scales[tok].to(tile.device)] = s.to(torch.uint8)


def fill(pages, seed, key=1.0, val=1.0):
    """Every slot of a pool with rounded normal keys and values."""
    n, n_kv, tiles, tb = pages.shape
    hd = tb // 17
    g = torch.Generator(device=pages.device).manual_seed(seed)
    pk, pv, sk, sv = places(hd, pages.device)
    for at in range(0, n, 64):
        some = pages[at:at + 64]
        for codes, scales, f in ((pk, sk, key), (pv, sv, val)):
            c, s = quantize(torch.randn(len(some), n_kv, tiles, 16, hd, generator=g, device=pages.device) * f)
            some[:, :, :, codes[:, 0::2]] = (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8)
            some[:, :, :, scales] = s.to(torch.uint8)


def turned(x, pos, freqs, amp, il):
    """(rotated x, sum of the magnitudes that each element is made of), in 64 bits."""
    x, r = x.double(), 2 * freqs.numel()
    t = pos.double()[:, None, None] * freqs
    c, s = t.cos() * amp, t.sin() * amp
    i, j = (slice(0, r, 2), slice(1, r, 2)) if il else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., i], x[..., j]
    y, m = x.clone(), x.abs()
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    m[..., i] = m[..., j] = (a.abs() + b.abs()) * amp
    return y, m


def normed(x, w, eps):
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def attention(q, pages, table, lengths, starts, first, scale):
    """(out, sum p |v| / sum p, largest scale sum |q k|, sum |v|) of every row in 64 bits; rows of no sequence NaN."""
    T, nh, hd = q.shape
    n_kv, cap = pages.shape[1], table.shape[1] * pages.shape[2] * 16
    out = torch.full((T, nh, hd), math.nan, dtype=torch.float64, device=q.device)
    mags, sums = torch.zeros_like(out), torch.zeros_like(out)
    tops = torch.zeros(T, nh, 1, dtype=torch.float64, device=q.device)
    edges = list(range(T + 1)) if starts is None else starts.tolist()
    for b, n in enumerate(lengths.tolist()):
        if edges[b + 1] <= edges[b]:
            continue
        k, v = rows_of(pages, table[b])
        gone = (table[b] < 0) | (table[b] >= pages.shape[0])
        gone = gone.repeat_interleave(pages.shape[2] * 16)
        for t in range(edges[b], edges[b + 1]):
            sees = 0 if n < 0 else min(max(n + first + t - edges[b], 0), cap)
            keep = (~gone[:sees]).nonzero()[:, 0]
            if not len(keep):
                out[t] = 0
                continue
            for h in range(n_kv):
                G = nh // n_kv
                qq, kk, vv = q[t, h * G:(h + 1) * G].double(), k[h, keep], v[h, keep]
                s = qq @ kk.T * scale
                p = torch.exp(s - s.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                out[t, h * G:(h + 1) * G] = p @ vv
                mags[t, h * G:(h + 1) * G] = p @ vv.abs()
                sums[t, h * G:(h + 1) * G] = vv.abs().sum(0)
                tops[t, h * G:(h + 1) * G] = (qq.abs() @ kk.abs().T * abs(scale)).amax(-1, keepdim=True)
    return out, mags, tops, sums
