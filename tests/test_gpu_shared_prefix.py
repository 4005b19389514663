"""shared_prefix_attn against attention in 64 bits.

Tolerance, for a row with A = the largest scale * sum |q_i k_i| of its keys and W = sum p |v|: a
score is a sum of hd products whose roundings (half a step, 2^-24, of partial sums up to A) are
independent, off by about 2^-24 sqrt(hd) A, four times that at most here; the exponent's reference
and scale 2 * 2^-24 A; the query's and the probability's 22 bits of fp16 caches 2^-23 each; exp2 and
the division some 2^-22; the sums over n keys 2 * 2^-24 sqrt(n):
  |error| <= 2^-24 ((4 sqrt(hd) + 4) A + 2 sqrt(n) + 16) W.
fp32 caches behind more than 64 rows add 2^-39 max |v|: a value there is the sum of two fp16 values of v 2^-E,
whose largest of 8 keys is at least 2^14; the low one's last place is 2^-24 at least (fp16's smallest),
so an element is off by up to 2^-25 2^E <= 2^-39 max |v| however small it is itself, and sum p = 1."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from pico_hip import kernels
    return kernels


def plain(q, kp, vp, ko, vo, P, own, scale=None):
    """(rows, their tolerances) in 64 bits, each sequence on its own."""
    B, nh, hd = q.shape
    nkv = kp.shape[0]
    scale = hd ** -0.5 if scale is None else scale
    out, tol = (torch.zeros(B, nh, hd, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        n = min(int(own[b]), ko.shape[2])
        if n < 0 or n + P == 0:
            continue
        for j in range(nkv):
            k = torch.cat([kp[j, :P], ko[b, j, :n]]).double()
            v = torch.cat([vp[j, :P], vo[b, j, :n]]).double()
            h = slice(j * (nh // nkv), (j + 1) * (nh // nkv))
            x = q[b, h].double()
            s = x @ k.T * scale
            p = torch.softmax(s, -1)
            A = abs(scale) * (x.abs() @ k.abs().T).amax(-1, keepdim=True)
            out[b, h] = p @ v
            tol[b, h] = 2.0 ** -24 * ((4 * math.sqrt(hd) + 4) * A + 2 * math.sqrt(P + n) + 16) * (p @ v.abs())
            if kp.dtype is torch.float32 and B * (nh // nkv) > 64:
                tol[b, h] += 2.0 ** -39 * v.abs().max()
    return out, tol


def make(seed, B, nh, nkv, hd, P, cap, dtype, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    q = r(B, nh, hd) * 1.5
    kp, vp = (r(nkv, P + extra, hd) * 1.2).to(dtype), r(nkv, P + extra, hd).to(dtype)
    ko, vo = (r(B, nkv, cap, hd) * 1.2).to(dtype), r(B, nkv, cap, hd).to(dtype)
    own = torch.randint(0, cap + 1, (B,), generator=g, device=DEV)
    return q, kp, vp, ko, vo, own


def close(got, ref, tol):
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - ref).abs() / tol.clamp_min(1e-30)).max()))


# one launch up to 640 (fp32) or 1280 keys (fp16), solo and shared rows beyond
SHAPES = [(1, 14, 2, 64, 1, 1), (3, 14, 2, 64, 1400, 64), (2, 28, 4, 128, 1281, 300), (1, 28, 4, 128, 3001, 1), (5, 25, 5, 64, 2500, 0),
          (20, 28, 4, 128, 1500, 70), (80, 16, 16, 64, 130, 129), (129, 14, 2, 64, 1290, 5), (260, 4, 1, 128, 33, 700), (1, 14, 2, 64, 33, 0), (4, 14, 2, 64, 277, 64), (3, 28, 4, 128, 129, 130), (16, 14, 2, 64, 1500, 40),
          (10, 28, 4, 128, 700, 33), (37, 28, 4, 128, 513, 9), (9, 25, 5, 64, 64, 200), (5, 16, 16, 64, 95, 31),
          (70, 12, 1, 64, 260, 3), (2, 64, 1, 128, 300, 300), (130, 4, 4, 64, 31, 5), (2, 8, 2, 128, 4097, 1000), (65, 2, 1, 64, 2000, 128),
          # several row tiles of a number of chunks that 8 does not divide
          (20, 15, 5, 64, 3000, 60), (50, 15, 5, 128, 2000, 33), (400, 3, 3, 64, 700, 20), (100, 9, 3, 128, 64, 900)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,nh,nkv,hd,P,cap", SHAPES)
def test_shared_prefix_attn(K, B, nh, nkv, hd, P, cap, dtype):
    q, kp, vp, ko, vo, own = make(B + P, B, nh, nkv, hd, P, cap, dtype)
    ref, tol = plain(q, kp, vp, ko, vo, P, own)
    got = K.shared_prefix_attn(q, kp, vp, ko, vo, own, round_fp16=False)
    close(got, ref, tol)
    assert torch.equal(K.shared_prefix_attn(q, kp, vp, ko, vo, own.int(), round_fp16=False), got)
    # rounded to fp16: half a step more
    close(K.shared_prefix_attn(q, kp, vp, ko, vo, own), ref, tol * (1 + 2 ** -11) + (ref.abs() * 2 ** -11).clamp_min(2 ** -25))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,extra", [(2, 100), (2, 1500), (40, 100), (40, 1500)])
def test_lengths_and_what_lies_behind_them(K, B, extra, hd, dtype):
    """Prefixes and own lengths of zero, one, around tiles and chunks, on the host and on the device;
    what lies behind a length may be NaN or infinite; negative lengths give zeros."""
    nh, nkv, cap = 4, 2, 300
    q, kp, vp, ko, vo, _ = make(hd + B, B, nh, nkv, hd, 0, cap, dtype, extra=extra)
    lengths = [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 300, 1000, -1, -7]
    own = torch.tensor([lengths[i % len(lengths)] for i in range(B)], device=DEV)
    for P in [n for n in (0, 1, 32, 100, 127, 128, 300, 513, 1500) if n <= extra]:
        for o in (own, own.roll(3), torch.zeros_like(own)):
            k1, v1, k2, v2 = kp.clone(), vp.clone(), ko.clone(), vo.clone()
            k1[:, P:], v1[:, P:] = float("nan"), math.inf
            for b in range(B):
                n = min(max(int(o[b]), 0), cap)
                k2[b, :, n:], v2[b, :, n:] = math.inf, float("nan")
            ref, tol = plain(q, kp, vp, ko, vo, P, o)
            got = K.shared_prefix_attn(q, k1, v1, k2, v2, o, prefix_len=P, round_fp16=False)
            close(got, ref, tol)
            dev = K.shared_prefix_attn(q, k1, v1, k2, v2, o - 5, prefix_len=torch.tensor(P, device=DEV), own_offset=5,
                                       round_fp16=False)
            close(dev, ref, tol)
            none = (o < 0) | ((o.clamp_min(0) + P) == 0)
            assert bool((got[none] == 0).all()) and bool((dev[none] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("P", [45, 1645])
def test_seen_infinity_at_the_end_of_a_tile(K, P, dtype):
    """The last key a row sees is copied behind the length; its infinite value counts once."""
    q, kp, vp, ko, vo, _ = make(3, 3, 4, 2, 64, P, 7, dtype)
    vp[1, P - 1, 5] = math.inf
    got = K.shared_prefix_attn(q, kp, vp, ko, vo, 3, round_fp16=False)
    assert not bool(torch.isfinite(got[:, 2:, 5]).any()) and bool(torch.isfinite(got[:, :2]).all())
    assert bool(torch.isfinite(got[:, 2:, :5]).all()) and bool(torch.isfinite(got[:, 2:, 6:]).all())
    if dtype is torch.float32:
        assert bool((got[:, 2:, 5] == math.inf).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,hd,P", [(3, 64, 400), (3, 64, 1700), (40, 128, 1700)])
def test_nan_keys_reach_the_rows_that_see_them(K, B, hd, P, dtype):
    q, kp, vp, ko, vo, own = make(B, B, 4, 2, hd, P, 40, dtype)
    clean = K.shared_prefix_attn(q, kp, vp, ko, vo, own)
    for lo, hi in ((5, 6), (128, 256), (32, 64)):
        bad = kp.clone()
        bad[1, lo:hi, 7] = float("nan")
        got = K.shared_prefix_attn(q, bad, vp, ko, vo, own)
        assert torch.equal(got[:, :2], clean[:, :2]) and bool(torch.isnan(got[:, 2:]).all())
    bad, own = ko.clone(), torch.full_like(own, 10)
    clean = K.shared_prefix_attn(q, kp, vp, ko, vo, own)
    bad[1, 0, 9, 3] = float("nan")
    got = K.shared_prefix_attn(q, kp, vp, bad, vo, own)
    assert bool(torch.isnan(got[1, :2]).all()) and torch.equal(got[1, 2:], clean[1, 2:])
    assert torch.equal(got[[0, 2]], clean[[0, 2]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,P", [(5, 300), (5, 1500), (40, 1500)])
@pytest.mark.parametrize("mag", [2.0 ** -30, 2.0 ** -12, 1.0, 30.0, 3000.0, 2.0 ** 40])
def test_magnitudes(K, mag, B, P, dtype):
    """Queries of any magnitude (scores from nothing to one key taking all), subnormal fp16 values."""
    q, kp, vp, ko, vo, own = make(1, B, 14, 2, 64, P, 30, dtype)
    q = q * mag
    vp[:, ::2] *= 2.0 ** -13
    vo[:, :, ::2] *= 2.0 ** -13
    scale = 0.125 if mag < 2.0 ** 30 else 2.0 ** -43
    ref, tol = plain(q, kp, vp, ko, vo, P, own, scale)
    got = K.shared_prefix_attn(q, kp, vp, ko, vo, own, scale=scale, round_fp16=False)
    close(got, ref, tol)


@pytest.mark.parametrize("scale", [-0.125, 0.0, 0.5])
@pytest.mark.parametrize("B,P", [(2, 100), (2, 1500), (40, 1500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_scales(K, scale, B, P, dtype):
    q, kp, vp, ko, vo, own = make(4, B, 14, 2, 64, P, 37, dtype)
    ref, tol = plain(q, kp, vp, ko, vo, P, own, scale)
    close(K.shared_prefix_attn(q, kp, vp, ko, vo, own, scale=scale, round_fp16=False), ref, tol)


@pytest.mark.parametrize("B", [2, 40])
def test_fp32_caches_of_any_magnitude(K, B):
    """Keys and values of fp32 range, groups of keys of very different ones, an infinite value."""
    q, kp, vp, ko, vo, own = make(6, B, 14, 2, 64, 1500, 20, torch.float32)
    kp[:, 300:600] *= 1e-6
    kp[:, 700:708] *= 3.0
    q[:, 2] *= 1e-20
    vp[:, 40:60] *= 1e30
    vp[:, 900:1400] *= 1e-25
    ref, tol = plain(q, kp, vp, ko, vo, 1500, own)
    close(K.shared_prefix_attn(q, kp, vp, ko, vo, own, round_fp16=False), ref, tol)
    kp, vp = kp * 1e18, torch.full_like(vp, 1e-30)
    ref, tol = plain(q, kp, vp, ko * 1e18, vo * 1e-30, 1500, own, 1e-19)
    close(K.shared_prefix_attn(q, kp, vp, ko * 1e18, vo * 1e-30, own, scale=1e-19, round_fp16=False), ref, tol)
    vp[0, 1000, 9] = math.inf
    got = K.shared_prefix_attn(q, kp, vp, ko * 1e18, vo * 1e-30, own, scale=1e-19, round_fp16=False)
    assert not bool(torch.isfinite(got[:, :7, 9]).any())
    got[:, :7, 9], ref[:, :7, 9] = 0, 0
    close(got, ref, tol)


def test_same_as_decode_attn(K):
    """One sequence: decode_attn over the two caches laid end to end."""
    for hd, nh, nkv, P, n in ((64, 14, 2, 700, 20), (128, 28, 4, 33, 100), (64, 14, 2, 50, 1)):
        q, kp, vp, ko, vo, _ = make(P, 1, nh, nkv, hd, P, n, torch.float32)
        ref, tol = plain(q, kp, vp, ko, vo, P, [n])
        want = K.decode_attn(q[0], torch.cat([kp, ko[0]], 1), torch.cat([vp, vo[0]], 1), round_fp16=False)
        got = K.shared_prefix_attn(q, kp, vp, ko, vo, n, round_fp16=False)[0]
        assert bool(((got - want).abs() <= 2 * tol[0]).all())


def test_deterministic_and_any_workspace(K):
    q, kp, vp, ko, vo, own = make(8, 20, 28, 4, 128, 3000, 77, torch.float16)
    a = K.shared_prefix_attn(q, kp, vp, ko, vo, own)
    ws = K.shared_prefix_attn_workspace(20, 28, 4, 128, 3000, 77, DEV)
    for fill in (0, 0xFF, 0x7F):
        ws.fill_(fill)
        assert torch.equal(K.shared_prefix_attn(q, kp, vp, ko, vo, own, workspace=ws), a)


def test_graphs_that_share_a_workspace_and_streams(K):
    """Two captured calls on one workspace, replayed in turn, read lengths and rows when replayed;
    calls on two streams with workspaces of their own."""
    B, nh, nkv, hd, P, cap = 6, 14, 2, 64, 900, 50
    q, kp, vp, ko, vo, own = make(1, B, nh, nkv, hd, P, cap, torch.float32)
    plen = torch.tensor([P], device=DEV)
    ws = K.shared_prefix_attn_workspace(B, nh, nkv, hd, P, cap, DEV)
    out1, out2 = torch.empty_like(q), torch.empty_like(q)
    q2 = q.flip(0).contiguous()
    K.shared_prefix_attn(q, kp, vp, ko, vo, own, plen, workspace=ws, out=out1)
    graphs = []
    for x, o in ((q, out1), (q2, out2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.shared_prefix_attn(x, kp, vp, ko, vo, own, plen, workspace=ws, out=o)
        graphs.append(g)
    for step in range(4):
        own.copy_(torch.arange(B, device=DEV) * 3 + step)
        plen.fill_(P - 100 * step)
        q.normal_()
        graphs[0].replay()
        graphs[1].replay()
        for x, o in ((q, out1), (q2, out2)):
            ref, tol = plain(x, kp, vp, ko, vo, P - 100 * step, own)
            close(o, ref, tol * (1 + 2 ** -11) + (ref.abs() * 2 ** -11).clamp_min(2 ** -25))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = K.shared_prefix_attn(q, kp, vp, ko, vo, own)
    with torch.cuda.stream(s2):
        b = K.shared_prefix_attn(q2, kp, vp, ko, vo, own)
    torch.cuda.synchronize()
    assert torch.equal(a, K.shared_prefix_attn(q, kp, vp, ko, vo, own))
    assert torch.equal(b, K.shared_prefix_attn(q2, kp, vp, ko, vo, own))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_long_cache_offsets(K, dtype):
    """Byte offsets past 32 bits: the last kv heads of long caches."""
    hd, nkv, P = 128, 5, 1 << 20
    q = torch.randn(2, nkv, hd, device=DEV)
    kp = torch.zeros(nkv, P, hd, device=DEV, dtype=dtype)     # 2.7 GB in fp32
    vp = torch.zeros_like(kp)
    kp[4, P - 40:] = torch.randn(40, hd, device=DEV).to(dtype) * 3
    vp[4, P - 40:] = torch.randn(40, hd, device=DEV).to(dtype)
    vp[:, :, 0] = 1.0
    ko = torch.randn(2, nkv, 3, hd, device=DEV).to(dtype)
    got = K.shared_prefix_attn(q * 4, kp, vp, ko, ko, 0, round_fp16=False)
    for b in range(2):
        s = kp[4, P - 40:].double() @ (q[b, 4] * 4).double() * hd ** -0.5
        e = torch.exp(s)
        want = e @ vp[4, P - 40:].double()
        want = want / (e.sum() + (P - 40))
        A = float((kp[4, P - 40:].double().abs() @ (q[b, 4] * 4).double().abs()).max()) * hd ** -0.5
        W = e @ vp[4, P - 40:].double().abs() / (e.sum() + (P - 40))
        tol = 2.0 ** -24 * ((4 * math.sqrt(hd) + 4) * A + 2 * math.sqrt(P) + 16) * W
        assert bool(((got[b, 4].double() - want).abs()[1:] <= tol[1:]).all())
        assert bool(((got[b, :4, 0] - 1).abs() <= 2.0 ** -24 * (2 * math.sqrt(P) + 16)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_long_cache_offsets_of_many_rows(K, dtype):
    """The same with row tiles that share the keys; fp32 values have the 2^-39 of their group's largest besides."""
    hd, nkv, P, B = 128, 5, 1 << 20, 70
    q = torch.randn(B, nkv, hd, device=DEV) * 4
    kp = torch.zeros(nkv, P, hd, device=DEV, dtype=dtype)
    vp = torch.zeros_like(kp)
    kp[4, P - 40:] = torch.randn(40, hd, device=DEV).to(dtype) * 3
    vp[4, P - 40:] = torch.randn(40, hd, device=DEV).to(dtype)
    vp[:, :, 0] = 1.0
    ko = torch.randn(B, nkv, 3, hd, device=DEV).to(dtype)
    got = K.shared_prefix_attn(q, kp, vp, ko, ko, 0, round_fp16=False)[:, 4].double()
    k, v, x = kp[4, P - 40:].double(), vp[4, P - 40:].double(), q[:, 4].double()
    s = x @ k.T * hd ** -0.5
    top = s.amax(1, keepdim=True).clamp_min(0)
    e, rest = torch.exp(s - top), torch.exp(-top) * (P - 40)
    total = e.sum(1, keepdim=True) + rest
    A = (x.abs() @ k.abs().T).amax(1, keepdim=True) * hd ** -0.5
    tol = 2.0 ** -24 * ((4 * math.sqrt(hd) + 4) * A + 2 * math.sqrt(P) + 16) * (e @ v.abs() / total) + 2.0 ** -39 * v.abs().max()
    assert bool(((got - e @ v / total).abs()[:, 1:] <= tol[:, 1:]).all())
    assert bool(((got[:, 0] - 1).abs() <= 2.0 ** -24 * (2 * math.sqrt(P) + 16)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_many_sequences(K, dtype):
    """Thousands of sequences: more workgroups than a round holds, of one chunk each."""
    B, n, hd, P, cap = 9001, 2, 64, 700, 2
    q, kp, vp, ko, vo, own = make(8, B, n, n, hd, P, cap, dtype)
    own[::7] = -1
    got = K.shared_prefix_attn(q, kp, vp, ko, vo, own, round_fp16=False).double()
    x, scale = q.double(), hd ** -0.5
    s = torch.cat([torch.einsum("bhd,hpd->bhp", x, kp.double()), torch.einsum("bhd,bhpd->bhp", x, ko.double())], -1) * scale
    A = scale * torch.cat([torch.einsum("bhd,hpd->bhp", x.abs(), kp.double().abs()),
                           torch.einsum("bhd,bhpd->bhp", x.abs(), ko.double().abs())], -1).amax(-1, keepdim=True)
    s[..., P:].masked_fill_(torch.arange(cap, device=DEV) >= own[:, None, None], -math.inf)
    p = torch.softmax(s, -1)
    out = lambda f: torch.einsum("bhp,hpd->bhd", p[..., :P], f(vp.double())) + torch.einsum("bhp,bhpd->bhd", p[..., P:], f(vo.double()))
    tol = 2.0 ** -24 * ((4 * math.sqrt(hd) + 4) * A + 2 * math.sqrt(P + cap) + 16) * out(torch.abs) + 2.0 ** -39 * 8
    live = own >= 0
    assert bool(((got - out(lambda v: v)).abs() <= tol)[live].all()) and bool((got[~live] == 0).all())


def test_refusals(K):
    q, kp, vp, ko, vo, own = make(1, 3, 4, 2, 64, 40, 8, torch.float32)
    bad = [(q[0], kp, vp, ko, vo, own), (q, kp.half(), vp, ko, vo, own), (q, kp, vp, ko.half(), vo.half(), own),
           (q, kp.double(), vp.double(), ko.double(), vo.double(), own), (q, kp[:, :, ::2], vp[:, :, ::2], ko, vo, own),
           (q, kp, vp[:, :9].contiguous(), ko, vo, own), (q, kp, vp, ko[:2], vo[:2], own), (q, kp, vp, ko[:, :1], vo[:, :1], own),
           (q, kp, vp, ko, vo, own[:2]), (q, kp, vp, ko, vo, own.float()), (q, kp, vp, ko, vo, own, 41), (q, kp, vp, ko, vo, own, -1),
           (q, kp, vp, ko, vo, own.cpu()), (q.cpu(), kp, vp, ko, vo, own), (q, kp, vp, ko, vo, own, torch.zeros(2, device=DEV).long()),
           (q[..., :32], kp, vp, ko, vo, own), (q, kp.transpose(1, 2).contiguous().transpose(1, 2), vp, ko, vo, own)]
    for args in bad:
        with pytest.raises(ValueError):
            K.shared_prefix_attn(*args)
    long = torch.zeros(2, 5000, 64, device=DEV)
    with pytest.raises(RuntimeError):    # too small a workspace
        K.shared_prefix_attn(q, long, long, ko, vo, own, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError):    # head sizes of 64 and 128
        K.shared_prefix_attn(*(t[..., :32].contiguous() for t in (q, kp, vp, ko, vo)), own)
    with pytest.raises(RuntimeError):    # whole groups
        K.shared_prefix_attn(q[:, :3], kp, vp, ko, vo, own)
    with pytest.raises(ValueError):
        K.shared_prefix_attn(q, kp, vp, ko, vo, own, out=torch.empty(3, 4, 64, device=DEV).half())
    assert K.shared_prefix_attn(q[:0], kp, vp, ko[:0], vo[:0], own[:0]).shape == (0, 4, 64)
