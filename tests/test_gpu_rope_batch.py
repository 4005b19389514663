"""rope_positions and rope_append against the rotation in 64 bits.

Tolerance of a rotated element: the rest of the angle, its conversion and the two series' roundings
leave at most 2^-22 amp on sine and cosine (2^-24.2 of angle, 2^-24 of evaluation, half steps of 2^-25
twice, 2^-28 of truncation), the two products and their sum 2^-24 each: under
2^-21 amp (|x| + |y|) in fp32; stored in fp16 half a step more, 2^-11 of the value (2^-25 at least)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from pico_hip import kernels
    return kernels


def turned(x, pos, freqs, amp, il):
    """(rotated x, sum of the magnitudes that each element is made of), in 64 bits."""
    x = x.double()
    r = 2 * freqs.numel()
    t = pos.double()[:, None, None] * freqs
    c, s = t.cos() * amp, t.sin() * amp
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if il else (x[..., :r // 2], x[..., r // 2:r])
    y, m = x.clone(), torch.zeros_like(x)
    both = (a.abs() + b.abs()) * amp
    if il:
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, a * s + b * c
        m[..., 0:r:2] = m[..., 1:r:2] = both
    else:
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, a * s + b * c
        m[..., :r // 2] = m[..., r // 2:r] = both
    return y, m


def close(got, ref, mags):
    tol = mags * 2.0 ** -21
    if got.dtype is torch.float16:
        tol = tol + (ref.abs() * 2.0 ** -11).clamp_min(2.0 ** -25)
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, at most {float((got.double() - ref).abs().max())}"


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("T,n,hd,rot", [(1, 1, 64, 64), (1, 14, 64, 64), (7, 3, 128, 64), (257, 16, 64, 64),
                                        (33, 5, 80, 20), (5, 2, 66, 22), (3, 4, 7, 6), (2, 1, 2, 2), (1000, 28, 128, 128),
                                        (4099, 2, 256, 256)])
def test_rope_positions(K, T, n, hd, rot, dtype, il):
    x = rand(T, T, n, hd).to(dtype)
    freqs, amp = K.rope_freqs(rot, 1e6)
    pos = torch.randint(-50, 5000, (T,), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    keep = x.clone()
    got = K.rope_positions(x, pos, freqs, interleaved=il)
    assert torch.equal(x, keep)
    ref, mags = turned(x, pos, freqs, amp, il)
    close(got, ref, mags)
    assert torch.equal(got[..., rot:], x[..., rot:])
    assert torch.equal(K.rope_positions(x, pos.int(), freqs, interleaved=il), got)
    assert K.rope_positions(x, pos, freqs, interleaved=il, out=x) is x and torch.equal(x, got)   # in place


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rope_positions_strides(K, dtype):
    """Heads first, rows inside wider ones, an unaligned start, one row for all tokens, a last dim apart."""
    freqs, amp = K.rope_freqs(32, 10000.0)
    pos = torch.arange(40, device=DEV) * 7
    wide = rand(2, 40, 6, 100).to(dtype)
    views = [rand(1, 6, 40, 64).to(dtype).transpose(0, 1), wide[:, :, 4:68], wide[:, 1:4, 3:67], wide[:, ::2, :64],
             wide[:1, :, :64].expand(40, 6, 64), rand(3, 40, 64, 6).to(dtype).transpose(1, 2)]
    for x in views:
        ref, mags = turned(x, pos, freqs, amp, False)
        close(K.rope_positions(x, pos, freqs), ref, mags)
    # into rows of a wider tensor: what lies beside them stays
    out = torch.full((40, 6, 100), 7.0, device=DEV, dtype=dtype)
    K.rope_positions(wide[:, :, :64], pos, freqs, out=out[:, :, 20:84])
    ref, mags = turned(wide[:, :, :64], pos, freqs, amp, False)
    close(out[:, :, 20:84], ref, mags)
    assert bool((out[:, :, :20] == 7).all()) and bool((out[:, :, 84:] == 7).all())
    heads = torch.empty(6, 40, 64, device=DEV, dtype=dtype).transpose(0, 1)
    K.rope_positions(wide[:, :, :64], pos, freqs, out=heads)
    close(heads, ref, mags)


@pytest.mark.parametrize("far", [0, 32768, 1 << 20, (1 << 31) + 5, -(1 << 24)])
def test_rope_positions_far(K, far):
    """Angles of far positions keep their precision: position 2^31's product with f_j in 64 bits is
    exact to 2^-21 turns of the reference itself; compared with whole-number phases instead."""
    f = [2.0 ** -j for j in range(1, 17)]     # whole binary fractions of a turn: exact phases
    freqs = torch.tensor([2 * math.pi * x for x in f], dtype=torch.float64, device=DEV)
    pos = torch.arange(100, device=DEV) * 37 + far
    x = rand(5, 100, 2, 32)
    phase = torch.stack([torch.remainder(pos, 1 << j).double() / (1 << j) for j in range(1, 17)], 1) * (2 * math.pi)
    c, s = phase.cos()[:, None], phase.sin()[:, None]
    a, b = x[..., :16].double(), x[..., 16:].double()
    ref = torch.cat([a * c - b * s, a * s + b * c], -1)
    mags = (a.abs() + b.abs()).repeat(1, 1, 2)
    # 2 pi f, its product with 2 / pi and that with the position are rounded to 64 bits: 3 * 2^-53 of the angle
    slack = abs(far) * math.pi * 2.0 ** -51
    got = K.rope_positions(x, pos, freqs)
    assert bool(((got.double() - ref).abs() <= mags * (2.0 ** -21 + slack)).all())


def test_rope_positions_against_differences(K):
    """Turning by p and then by -p gives x back; turning by p + d is turning by p, then by d."""
    freqs, _ = K.rope_freqs(64, 1e6)
    x, p, d = rand(1, 50, 4, 64), torch.arange(50, device=DEV) * 31, torch.full((50,), 777, device=DEV)
    y = K.rope_positions(x, p, freqs)
    m = (x[..., :32].abs() + x[..., 32:].abs()).repeat(1, 1, 2).double()
    assert bool(((K.rope_positions(y, -p, freqs) - x).double().abs() <= m * 2 ** -19).all())
    assert bool(((K.rope_positions(y, d, freqs) - K.rope_positions(x, p + d, freqs)).double().abs() <= m * 2 ** -19).all())


@pytest.mark.parametrize("cache", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,nh,nkv,hd,rot,il,cap", [(1, 14, 2, 64, 64, False, 9), (5, 28, 4, 128, 128, False, 17),
                                                    (33, 4, 4, 64, 20, True, 3), (3, 12, 1, 80, 40, True, 5),
                                                    (2, 2, 1, 6, 2, False, 1), (300, 25, 5, 64, 32, False, 2)])
def test_rope_append(K, B, nh, nkv, hd, rot, il, cap, cache):
    g = torch.Generator(device=DEV).manual_seed(B)
    freqs, amp = K.rope_freqs(rot, 1e6, scaling="yarn", factor=4.0, original_context=4096)
    qkv = rand(B, B, (nh + 2 * nkv) * hd)
    k, v = (torch.full((B, nkv, cap, hd), float("nan"), device=DEV, dtype=cache) for _ in range(2))
    slots = torch.randint(-1, cap + 1, (B,), generator=g, device=DEV)    # some outside
    slots[0] = cap - 1
    pos = slots + 6000
    q = K.rope_append(qkv, pos, freqs, nh, k, v, slot_offset=-6000, amp=amp, interleaved=il)
    rows = qkv.view(B, nh + 2 * nkv, hd)
    ref, mags = turned(rows[:, :nh + nkv], pos, freqs, amp, il)
    close(q, ref[:, :nh], mags[:, :nh])
    for b, s in enumerate(slots.tolist()):
        inside = 0 <= s < cap
        others = [i for i in range(cap) if i != s]
        assert bool(torch.isnan(k[b, :, others]).all()) and bool(torch.isnan(v[b, :, others]).all())
        if inside:
            close(k[b, :, s], ref[b, nh:], mags[b, nh:])
            assert torch.equal(v[b, :, s], rows[b, nh + nkv:].to(cache))


def test_rope_append_tables_and_strided_rows(K):
    """(cos, sin) tables read at the positions, rows inside wider ones, positions past the table."""
    B, nh, nkv, hd = 6, 4, 2, 64
    cos, sin = rand(1, 50, 32), rand(2, 50, 32)
    wide = rand(3, B, 600)
    qkv = wide[:, 8:8 + 8 * 64]
    pos = torch.tensor([0, 49, 7, 60, -3, 20], device=DEV, dtype=torch.int32)
    k, v = (torch.zeros(B, nkv, 100, hd, device=DEV) for _ in range(2))
    q = K.rope_append(qkv, pos, (cos, sin), nh, k, v, amp=1.5)
    x = qkv.reshape(B, 8, hd).double()
    at = pos.long().clamp(0, 49)
    c, s = cos[at].double()[:, None] * 1.5, sin[at].double()[:, None] * 1.5
    a, b = x[..., :32], x[..., 32:]
    ref = torch.cat([a * c - b * s, a * s + b * c], -1)
    mags = (a.abs() + b.abs()).repeat(1, 1, 2) * 1.5 * 4.5   # tables of normal values: under 4.5
    close(q, ref[:, :nh], mags[:, :nh])
    for i, p in enumerate(pos.tolist()):
        if p >= 0:
            close(k[i, :, p], ref[i, nh:nh + nkv], mags[i, nh:nh + nkv])
    assert bool((k[4] == 0).all()) and bool((v[4] == 0).all())
    # rows that are not 16-byte aligned: the same values
    q2 = K.rope_append(wide[:, 9:9 + 8 * 64], pos, (cos, sin), nh, k.clone(), v.clone())
    q3 = K.rope_append(wide[:, 9:9 + 8 * 64].contiguous(), pos, (cos, sin), nh, k.clone(), v.clone())
    assert torch.equal(q2, q3)


def test_rope_graph_and_stream(K):
    """A captured step reads its positions when it is replayed; a call on another stream."""
    B, nh, nkv, hd = 3, 14, 2, 64
    freqs, _ = K.rope_freqs(hd, 1e6)
    qkv, pos = rand(1, B, 18 * 64), torch.zeros(B, dtype=torch.int64, device=DEV)
    k, v = (torch.zeros(B, nkv, 20, hd, device=DEV) for _ in range(2))
    q = torch.empty(B, nh, hd, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.rope_append(qkv, pos, freqs, nh, k, v, out=q)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.rope_append(qkv, pos, freqs, nh, k, v, out=q)
    for step in range(4):
        pos.copy_(torch.arange(B, device=DEV) + 5 * step)
        qkv.normal_()
        graph.replay()
        k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
        want = K.rope_append(qkv, pos, freqs, nh, k2, v2)
        assert torch.equal(q, want)
        for b in range(B):
            assert torch.equal(k[b, :, b + 5 * step], k2[b, :, b + 5 * step])


def test_rope_empty_and_refusals(K):
    freqs, _ = K.rope_freqs(64)
    p = torch.zeros(3, dtype=torch.int64, device=DEV)
    x = rand(0, 3, 2, 64)
    assert K.rope_positions(x[:0], p[:0], freqs).shape == (0, 2, 64)
    k = torch.zeros(3, 1, 4, 64, device=DEV)
    assert K.rope_append(rand(0, 0, 256), p[:0], freqs, 2, k[:0], k[:0]).shape == (0, 2, 64)
    bad = [(x.double(), p, freqs), (x[0], p, freqs), (x, p[:2], freqs), (x, p.float(), freqs), (x, p, freqs.float()),
           (x[..., :62], p, freqs), (x, p.cpu(), freqs), (x.cpu(), p, freqs)]
    for args in bad:
        with pytest.raises(ValueError):
            K.rope_positions(*args)
    with pytest.raises(ValueError):
        K.rope_positions(x, p, freqs, out=x.half())
    with pytest.raises(RuntimeError):   # rows of the output that share memory
        K.rope_positions(x, p, freqs, out=torch.empty(2, 64, device=DEV).expand(3, 2, 64))
    qkv = rand(0, 3, 256)
    for args in [(qkv.half(), p, freqs, 2, k, k), (qkv, p, freqs, 3, k, k), (qkv, p, freqs, 2, k.double(), k.double()),
                 (qkv, p, freqs, 2, k, k.half()), (qkv, p, freqs, 2, k[:, :, ::2], k[:, :, ::2]),
                 (qkv, p, freqs, 2, k[:2], k[:2]), (qkv, p, (freqs, freqs), 2, k, k)]:
        with pytest.raises(ValueError):
            K.rope_append(*args)
