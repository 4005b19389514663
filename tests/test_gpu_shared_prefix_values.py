"""shared_prefix_attn with fp32 caches whose keys and values lie far apart, behind many rows and few, against
attention in 64 bits.

Tolerance, per row and dim, with p the probabilities, A_k = scale * sum |q_i k_i| of key k, o the result:
* scores: a sum of hd products whose roundings (2^-24 of partial sums up to A_k) are independent, four times
  2^-24 sqrt(hd) A_k at most here, the reference and scale 4 * 2^-24 A_k, the query's and the key's 22 bits
  2 * 2^-23 A_k; a changed score d_k moves the result by p_k d_k (v_k - o):
  2^-24 (4 sqrt(hd) + 8) sum p_k A_k (|v_k| + |o|);
* exp2, the division, 22 bits of probability and value, sums over n keys: 2^-24 (2 sqrt(n) + 20) W, W = sum p |v|;
* behind more than 64 rows, by groups of 8 keys from the prefix's start with G the largest magnitude of a group: a value's two
  parts end at 2^-39 G, and only groups in which every four neighbouring dims of a key hold 2^-14 G (or
  zeros) are taken that way, so 2^-25 sum p c, c the largest of an element's four neighbours; a
  probability's end at 2^-25 where the largest p G of a row stands for 2^8 2^14 at least, so
  2^-32 max(p G) sum |v| / G, over keys with G <= 2^14 c alone;
* with fp16 caches a probability ends at 2^-33 of the row's largest one: 2^-33 max(p) sum |v|.
Nothing in it grows with a value that has no weight."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from pico_hip import kernels
    return kernels


def plain(q, kp, vp, ko, vo, own, scale):
    """(rows, their tolerances) in 64 bits."""
    B, nh, hd = q.shape
    nkv, P, _ = kp.shape
    group = nh // nkv
    out, tol = (torch.zeros(B, nh, hd, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        n = int(own[b])
        for j in range(nkv):
            k = torch.cat([kp[j], ko[b, j, :n]]).double()
            v = torch.cat([vp[j], vo[b, j, :n]]).double()
            h = slice(j * group, (j + 1) * group)
            x = q[b, h].double()
            p = torch.softmax(x @ k.T * scale, -1)
            A = abs(scale) * (x.abs() @ k.abs().T)
            o = p @ v
            W = p @ v.abs()
            t = 2.0 ** -24 * (4 * math.sqrt(hd) + 8) * ((p * A) @ v.abs() + (p * A).sum(-1, keepdim=True) * o.abs())
            t += 2.0 ** -24 * (2 * math.sqrt(P + n) + 20) * W
            if kp.dtype is torch.float16:
                t += 2.0 ** -33 * p.amax(-1, keepdim=True) * v.abs().sum(0)
            elif B * group > 64:
                w = torch.nn.functional.pad(vp[j].double().abs(), (0, 0, 0, -P % 8)).view(-1, 8, hd)
                G = w.amax((1, 2))[:, None].expand(-1, 8).reshape(-1)[:P]
                c = vp[j].double().abs().view(P, hd // 4, 4).amax(-1, keepdim=True).expand(-1, -1, 4).reshape(P, hd)
                t += 2.0 ** -25 * p[:, :P] @ c
                least = torch.where(c > 0, c, torch.full_like(c, math.inf)).amin(1)
                most = torch.minimum(G, 2.0 ** 14 * least.nan_to_num(posinf=0.0))
                t += 2.0 ** -32 * (p[:, :P] * most).amax(-1, keepdim=True) * (vp[j].double().abs() / G.clamp_min(1e-300)[:, None]).sum(0)
            out[b, h], tol[b, h] = o, t
    return out, tol


def make(seed, B, hd, P, cap):
    """Queries whose first element is 4, so that a key's first element says how much weight it gets."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    nh, nkv = (14, 2) if hd == 64 else (21, 3)
    q = r(B, nh, hd) * 1.2
    q[..., 0] = 4.0
    return q, r(nkv, P, hd), r(nkv, P, hd), r(B, nkv, cap, hd), r(B, nkv, cap, hd), torch.randint(0, cap + 1, (B,), generator=g, device=DEV)


def check(K, q, kp, vp, ko, vo, own, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ref, tol = plain(q, kp, vp, ko, vo, own, scale)
    got = K.shared_prefix_attn(q, kp, vp, ko, vo, own, scale=scale, round_fp16=False)
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), (int((~(off <= tol)).sum()), float((off / tol).nan_to_num(math.inf).max()))
    return got


SHAPES = [(5, 64), (40, 64), (37, 128)]      # up to 64 rows of a kv head, and more


@pytest.mark.parametrize("B,hd", SHAPES)
@pytest.mark.parametrize("factor", [1e4, 1e6, 2.0 ** 30, 1e10, 2.0 ** 40, 1e25])
@pytest.mark.parametrize("rows", [(800, 808), (801, 802), (3, 5), (1535, 1536)])
def test_large_values_without_weight(K, rows, factor, B, hd):
    """Values far above the others in keys whose scores give them nothing: groups of 8 keys, single keys, the
    first and the last ones. The others keep their bits."""
    q, kp, vp, ko, vo, own = make(1, B, hd, 1536, 20)
    kp[:, slice(*rows), 0] = -60.0 * hd ** 0.5            # 240 nats under the others
    vp[:, slice(*rows)] *= factor
    check(K, q, kp, vp, ko, vo, own)


@pytest.mark.parametrize("B,hd", SHAPES)
@pytest.mark.parametrize("factor", [1e4, 1e10, 1e25])
def test_large_values_with_little_weight(K, factor, B, hd):
    """Their share is about that of the others together."""
    q, kp, vp, ko, vo, own = make(2, B, hd, 1300, 9)
    kp[:, 640:643, 0] = -(math.log(factor) / 4) * hd ** 0.5
    kp[:, 640:643, 1:] = 0
    vp[:, 640:643] *= factor
    check(K, q, kp, vp, ko, vo, own)


@pytest.mark.parametrize("B,hd", SHAPES)
@pytest.mark.parametrize("factor", [1e4, 1e10])
def test_small_values_with_all_the_weight(K, factor, B, hd):
    """A key that takes nearly everything, its value far under the others' or nothing."""
    for f in (1 / factor, 0.0):
        q, kp, vp, ko, vo, own = make(3, B, hd, 1536, 5)
        kp[:, 77, 0] = 2.5 * hd ** 0.5                    # e^10 times the others
        vp[:, 77] *= f
        check(K, q, kp, vp, ko, vo, own)


@pytest.mark.parametrize("B,hd", SHAPES)
@pytest.mark.parametrize("factor", [1e3, 1e6, 1e10])
def test_keys_far_apart(K, factor, B, hd):
    """Keys far above the others that point away from every query; queries with one such element that
    meets zeros."""
    q, kp, vp, ko, vo, own = make(4, B, hd, 1536, 20)
    kp[:, 900, :] *= 0.01 * factor
    kp[:, 900, 0] = -100.0 * factor
    check(K, q, kp, vp, ko, vo, own)
    q, kp, vp, ko, vo, own = make(5, B, hd, 1536, 20)
    q[..., 9] *= factor
    kp[..., 9] = 0
    ko[..., 9] = 0
    check(K, q, kp, vp, ko, vo, own)


@pytest.mark.parametrize("B,hd", SHAPES)
@pytest.mark.parametrize("dims", [slice(5, 6), slice(0, None, 4), slice(16, 48)])
@pytest.mark.parametrize("factor", [1e4, 1e8, 1e12])
def test_channels_far_apart(K, factor, dims, B, hd):
    """Dims of the values far above the others, in every key: those with other neighbours keep their bits."""
    q, kp, vp, ko, vo, own = make(6, B, hd, 1400, 20)
    vp[..., dims] *= factor
    vo[..., dims] *= factor
    scale = hd ** -0.5
    ref, _ = plain(q, kp, vp, ko, vo, own, scale)
    vs, os = vp.clone(), vo.clone()
    vs[..., dims] = 0
    os[..., dims] = 0
    got = check(K, q, kp, vp, ko, vo, own)
    # without the large dims in the bound, wherever none of an element's four neighbours is one
    _, tol = plain(q, kp, vs, ko, os, own, scale)
    off = (got.double() - ref).abs() > tol
    large = torch.zeros(hd, dtype=torch.bool, device=DEV)
    large[dims] = True
    off[..., large.view(-1, 4).any(1, keepdim=True).expand(-1, 4).reshape(-1)] = False
    assert not bool(off.any()), int(off.sum())


@pytest.mark.parametrize("B,hd", SHAPES)
def test_magnitudes_across_the_prefix(K, B, hd):
    """Stretches of keys whose values lie up to 2^180 apart, none of which has all the weight, and zeros."""
    q, kp, vp, ko, vo, own = make(7, B, hd, 2000, 20)
    vp[:, :500] *= 1e-26
    vp[:, 504:511] = 0
    vp[:, 700:1000] *= 1e-9
    kp[:, 1000:1200, 0] -= 30 * hd ** 0.5
    vp[:, 1000:1200] *= 1e28
    vp[:, 1600:] = 0
    check(K, q, kp, vp, ko, vo, own)
    vp[:] = 0
    vo[:] = 0
    assert bool((check(K, q, kp, vp, ko, vo, own) == 0).all())


@pytest.mark.parametrize("B,hd", SHAPES)
def test_infinities(K, B, hd):
    """An infinite value makes its dim infinite; an infinite key gives no weight or NaN by the query's sign; a
    key of minus infinity in the element where all queries are positive is no key."""
    q, kp, vp, ko, vo, own = make(8, B, hd, 1536, 20)
    clean, tol = plain(q, kp, vp, ko, vo, own, hd ** -0.5)
    group = q.shape[1] // kp.shape[0]
    bad = vp.clone()
    bad[1, 700, 9] = math.inf
    got = K.shared_prefix_attn(q, kp, bad, ko, vo, own, round_fp16=False)
    rows = slice(group, 2 * group)
    assert bool((got[:, rows, 9] == math.inf).all())
    got[:, rows, 9] = clean[:, rows, 9].float()
    tol[:, rows, 9] += 2.0 ** -23 * clean[:, rows, 9].abs()
    assert bool(((got.double() - clean).abs() <= tol).all())
    bad = kp.clone()
    bad[0, 33, 5] = math.inf
    got = K.shared_prefix_attn(q, bad, vp, ko, vo, own, round_fp16=False)
    up = q[:, :group, 5] > 0
    assert bool(torch.isnan(got[:, :group][up]).all()) and bool(torch.isfinite(got[:, :group][~up]).all())
    bad = kp.clone()
    bad[:, 1400:1430, 0] = -math.inf
    rest = torch.cat([kp[:, :1400], kp[:, 1430:]], 1), torch.cat([vp[:, :1400], vp[:, 1430:]], 1)
    ref, tol = plain(q, *rest, ko, vo, own, hd ** -0.5)
    got = K.shared_prefix_attn(q, bad, vp, ko, vo, own, round_fp16=False)
    assert bool(((got.double() - ref).abs() <= tol).all())


def test_rows_do_not_depend_on_the_batch(K):
    """A sequence behind few others and behind many: the same result within both tolerances, whatever the values."""
    q, kp, vp, ko, vo, own = make(9, 40, 64, 1536, 20)
    kp[:, 100:108, 0] = -480.0
    vp[:, 100:108] *= 2.0 ** 34
    few = check(K, q[:5], kp, vp, ko[:5], vo[:5], own[:5])
    many = check(K, q, kp, vp, ko, vo, own)
    _, tol = plain(q[:5], kp, vp, ko[:5], vo[:5], own[:5], 0.125)
    assert bool(((few - many[:5]).double().abs() <= 2 * tol + 2.0 ** -27).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("P", [300, 1500])
@pytest.mark.parametrize("B,hd", SHAPES)
def test_largest_queries(K, B, hd, P, dtype):
    """Queries near the end of fp32's range, which the scale brings back."""
    q, kp, vp, ko, vo, own = make(10, B, hd, P, 20)
    kp, vp, ko, vo = (t.to(dtype) for t in (kp, vp, ko, vo))
    for e in (110, 119, 120, 121, 124):
        check(K, q * 2.0 ** e, kp, vp, ko, vo, own, scale=2.0 ** (-3 - e))


@pytest.mark.parametrize("P", [300, 1500])
@pytest.mark.parametrize("B,hd", SHAPES)
def test_small_queries_with_huge_keys(K, B, hd, P):
    """Factors of the scores that leave fp32's range one by one and not together."""
    q, kp, vp, ko, vo, own = make(11, B, hd, P, 20)
    for qe, ke, se in ((-90, 118, -31), (-60, 100, -43), (-95, 60, 32)):
        check(K, q * 2.0 ** qe, kp * 2.0 ** ke, vp, ko * 2.0 ** ke, vo, own, scale=2.0 ** se)


def test_scales_that_are_no_numbers(K):
    q, kp, vp, ko, vo, own = make(12, 5, 64, 1500, 20)
    for x in (math.nan, math.inf, -math.inf):
        with pytest.raises(ValueError):
            K.shared_prefix_attn(q, kp, vp, ko, vo, own, scale=x)


def test_uneven_values_in_a_graph(K):
    """A captured call meets even and uneven keys and values in turn, and a prefix of any length; every replay is the
    eager call's result."""
    q, kp, vp, ko, vo, own = make(13, 37, 128, 1536, 20)
    plen = torch.tensor([1536], device=DEV)
    out = torch.empty_like(q)
    K.shared_prefix_attn(q, kp, vp, ko, vo, own, plen, round_fp16=False, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.shared_prefix_attn(q, kp, vp, ko, vo, own, plen, round_fp16=False, out=out)
    clean = kp.clone(), vp.clone()
    for n, factor in ((1536, 1.0), (1536, 1e9), (1000, 1e9), (1536, 1.0), (801, 1e9), (7, 1.0), (1536, math.inf), (1536, 1.0)):
        kp.copy_(clean[0])
        vp.copy_(clean[1])
        plen.fill_(n)
        kp[:, 800, 0] = -60.0 * 128 ** 0.5
        if math.isinf(factor):
            kp[:, 800, 0] = -math.inf
        else:
            vp[:, 800] *= factor
        graph.replay()
        got = out.clone()
        assert torch.equal(got, K.shared_prefix_attn(q, kp, vp, ko, vo, own, plen, round_fp16=False))
        assert torch.equal(got, K.shared_prefix_attn(q, kp, vp, ko, vo, own, plen, round_fp16=False))
        if not math.isinf(factor):
            ref, tol = plain(q, kp[:, :n], vp[:, :n], ko, vo, own, 128 ** -0.5)
            assert bool(((got.double() - ref).abs() <= tol).all())
        else:
            assert bool(torch.isfinite(got).all())
