"""qk_norm_rope against the norm and the rotation in 64 bits.

Tolerance of an element: the squares' sum is rounded at most 22 times (16 products in a lane, 6 joins), half of which
reaches the root, its mean, eps, root and quotient 4 times, the two products twice: under 2^-20 of the normed
element. The rotation as in rope_positions: under 2^-21 of the magnitudes that an element is made of. Stored in fp16
half a step more, 2^-11 of the value (2^-25 at least)."""

import pytest
import torch

from kv4_ref import normed, turned

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from pico_hip import kernels
    return kernels


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def close(got, x, w, pos, freqs, amp, il, eps):
    ref = x.double() if w is None else normed(x, w, eps)
    ref, mags = turned(ref, pos, freqs, amp, il)
    tol = mags * (2.0 ** -20 + 2.0 ** -21)
    if got.dtype is torch.float16:
        tol = tol + (ref.abs() * 2.0 ** -11).clamp_min(2.0 ** -25)
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, at most {float(err.max())}"


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("T,n,m,hd,rot", [(1, 28, 4, 128, 128), (1, 14, 2, 64, 64), (7, 3, 5, 128, 64), (257, 16, 16, 64, 64),
                                          (33, 5, 1, 80, 20), (5, 2, 3, 66, 22), (3, 4, 1, 7, 6), (2, 1, 1, 2, 2),
                                          (700, 32, 8, 128, 128), (65, 3, 2, 256, 256), (3, 2, 2, 512, 128), (4, 2, 1, 300, 298),
                                          (2, 2, 1, 511, 2), (9, 4, 2, 96, 96)])
def test_qk_norm_rope(K, T, n, m, hd, rot, dtype, il):
    q, k = (rand(1, T, n, hd) * 2).to(dtype), (rand(2, T, m, hd) * 0.1).to(dtype)
    wq, wk = 1 + rand(3, hd) * 0.3, 1 + rand(4, m, hd) * 0.3        # one weight for all heads, one each
    freqs, amp = K.rope_freqs(rot, 1e6)
    pos = torch.randint(-50, 60000, (T,), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    a, b = K.qk_norm_rope(q, k, wq, wk, pos, freqs, eps=1e-5, amp=1.25, interleaved=il)
    close(a, q, wq, pos, freqs, 1.25, il, 1e-5)
    close(b, k, wk, pos, freqs, 1.25, il, 1e-5)
    again = K.qk_norm_rope(q, k, wq, wk, pos.int(), freqs, eps=1e-5, amp=1.25, interleaved=il)
    assert torch.equal(again[0], a) and torch.equal(again[1], b)
    # a side without a weight is not normed, q alone, in place
    a2, b2 = K.qk_norm_rope(q, k, None, wk, pos, freqs, eps=1e-5, interleaved=il)
    close(a2, q, None, pos, freqs, 1.0, il, 1e-5)
    alone, none = K.qk_norm_rope(q, None, wq, None, pos, freqs, eps=1e-5, amp=1.25, interleaved=il)
    assert none is None and torch.equal(alone, a)
    out = K.qk_norm_rope(q, k, wq, wk, pos, freqs, eps=1e-5, amp=1.25, interleaved=il, out=(q, k))
    assert out[0] is q and torch.equal(q, a) and torch.equal(k, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides(K, dtype):
    """Rows of a fused projection, heads first, an unaligned start, a last dim apart, one row for all tokens."""
    freqs, _ = K.rope_freqs(64, 10000.0)
    pos = torch.arange(40, device=DEV) * 11
    w = 1 + rand(9, 64) * 0.2
    fused = rand(1, 40, (6 + 4) * 64 + 8).to(dtype)
    views = [(fused[:, :384].view(40, 6, 64), fused[:, 384:512].view(40, 2, 64)),
             (fused[:, 3:387].view(40, 6, 64), fused[:, 5:133].view(40, 2, 64)),
             (rand(2, 6, 40, 64).to(dtype).transpose(0, 1), rand(3, 2, 40, 64).to(dtype).transpose(0, 1)),
             (rand(4, 40, 64, 6).to(dtype).transpose(1, 2), rand(5, 40, 64, 2).to(dtype).transpose(1, 2)),
             (fused[:1, :384].view(1, 6, 64).expand(40, 6, 64), fused[:, :64].view(40, 1, 64))]
    for q, k in views:
        a, b = K.qk_norm_rope(q, k, w, w, pos, freqs)
        close(a, q, w, pos, freqs, 1.0, False, 1e-6)
        close(b, k, w, pos, freqs, 1.0, False, 1e-6)
        # into rows of something wider, whose single elements are summed in another order
        wide = torch.full((40, 9, 70), 7.0, device=DEV, dtype=dtype)
        K.qk_norm_rope(q, k, w, w, pos, freqs, out=(wide[:, :6, 2:66], wide[:, 6:6 + k.shape[1], 2:66]))
        close(wide[:, :6, 2:66], q, w, pos, freqs, 1.0, False, 1e-6)
        close(wide[:, 6:6 + k.shape[1], 2:66], k, w, pos, freqs, 1.0, False, 1e-6)
        assert bool((wide[:, :, :2] == 7).all()) and bool((wide[:, :, 66:] == 7).all()) and bool((wide[:, 8:] == 7).all())


def test_values(K):
    """Zero heads, an infinite element and NaN stay in their own head."""
    freqs, _ = K.rope_freqs(64, 10000.0)
    q = rand(1, 5, 3, 64)
    q[0, 0], q[1, 1, 7], q[2, 2, 40] = 0, float("inf"), float("nan")
    pos = torch.arange(5, device=DEV)
    a, _ = K.qk_norm_rope(q, None, torch.ones(64, device=DEV), None, pos, freqs)
    assert bool((a[0, 0] == 0).all()) and bool(a[2, 2].isnan().all())
    ok = torch.ones(5, 3, dtype=torch.bool, device=DEV)
    ok[1, 1] = ok[2, 2] = False
    assert bool(a[ok].isfinite().all())


def test_empty_and_refused(K):
    freqs, _ = K.rope_freqs(64, 10000.0)
    w = torch.ones(64, device=DEV)
    q, k = rand(1, 0, 3, 64), rand(1, 0, 1, 64)
    a, b = K.qk_norm_rope(q, k, w, w, torch.empty(0, device=DEV, dtype=torch.int64), freqs)
    assert a.shape == (0, 3, 64) and b.shape == (0, 1, 64)
    q, k, pos = rand(1, 4, 3, 64), rand(1, 4, 1, 64), torch.arange(4, device=DEV)
    bad = [lambda: K.qk_norm_rope(q.double(), k.double(), w, w, pos, freqs), lambda: K.qk_norm_rope(q, k.half(), w, w, pos, freqs),
           lambda: K.qk_norm_rope(q, k[:3], w, w, pos, freqs), lambda: K.qk_norm_rope(q, k, w[:32], w, pos, freqs),
           lambda: K.qk_norm_rope(q, k, w.half(), w, pos, freqs), lambda: K.qk_norm_rope(q, k, w, w, pos[:3], freqs),
           lambda: K.qk_norm_rope(q, k, w, w, pos, freqs.float()), lambda: K.qk_norm_rope(q, k, w, w, pos.cpu(), freqs),
           lambda: K.qk_norm_rope(q, k, w, w, pos, freqs, out=(q, None)),
           lambda: K.qk_norm_rope(q, k, w, w, pos, freqs, out=(q.half(), k)),
           lambda: K.qk_norm_rope(q, k, w, w, pos, K.rope_freqs(128)[0]),
           lambda: K.qk_norm_rope(rand(1, 2, 2, 520), None, None, None, pos[:2], freqs)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")


def test_another_stream_and_graph(K):
    freqs, _ = K.rope_freqs(64, 10000.0)
    w = 1 + rand(9, 64) * 0.2
    q, k, pos = rand(1, 33, 6, 64), rand(2, 33, 2, 64), torch.arange(33, device=DEV)
    want = K.qk_norm_rope(q, k, w, w, pos, freqs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = K.qk_norm_rope(q, k, w, w, pos, freqs)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            a, b = K.qk_norm_rope(q, k, w, w, pos, freqs)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for step in range(3):
        pos.add_(100)
        q.mul_(1.5)
        want = K.qk_norm_rope(q, k, w, w, pos, freqs)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]), step


def test_many_rows(K):
    """Rows beyond 2^25, single elements a lane: a wave takes a row of one short head."""
    T, w = (1 << 25) + 37, torch.tensor([1.0, 1.25], device=DEV)
    q = (rand(1, T, 1, 2) * 2).half()
    pos = torch.arange(T, device=DEV, dtype=torch.int32) % 5000
    freqs, _ = K.rope_freqs(2, 10000.0)
    a, _ = K.qk_norm_rope(q, None, w, None, pos, freqs, eps=1e-5)
    for at in (slice(0, 3000), slice((1 << 25) - 2000, T)):
        close(a[at], q[at], w, pos[at], freqs, 1.0, False, 1e-5)
    assert bool(a.isfinite().all())
