"""adjust_logits against its rules in 64 bits.

Tolerance: five fp32 operations at most (bias, repetition, frequency's product, two differences),
each off by half a step, 2^-24 of its result: 5 * 2^-24 of the largest value on the way. Stored in fp16
half a step more, 2^-11 of the value (2^-25 at least). Every sum keeps its sign when it is rounded, so
no case distinction goes another way."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from pico_hip import kernels
    return kernels


def plain(x, history, lengths, prompt, rules, bias, mask):
    """(adjusted logits, the largest magnitude on the way) of every element."""
    B, V = x.shape
    out, top = torch.empty(B, V, dtype=torch.float64), torch.empty(B, V, dtype=torch.float64)
    for b in range(B):
        z = x[b].double().cpu()
        if bias is not None:
            z = z + (bias if bias.dim() == 1 else bias[b if bias.shape[0] > 1 else 0]).double().cpu()
        big = z.abs()
        count, seen = torch.zeros(V, dtype=torch.float64), torch.zeros(V, dtype=torch.bool)
        if history is not None:
            ids = history[b].cpu()
            ids = ids[:max(0, min(int(lengths[b]), ids.numel()))] if lengths is not None else ids
            ids = ids[(ids >= 0) & (ids < V)].long()
            count += torch.bincount(ids, minlength=V)
            seen |= count > 0
        if prompt is not None:
            ids = (prompt if prompt.dim() == 1 else prompt[b if prompt.shape[0] > 1 else 0]).cpu()
            seen[ids[(ids >= 0) & (ids < V)].long()] = True
        rep, freq, pres = (float(torch.tensor(r, dtype=torch.float32)) if not isinstance(r, torch.Tensor) else float(r[b])
                           for r in rules)
        z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
        big = torch.maximum(big, z.abs())
        z = z - freq * count
        big = torch.maximum(torch.maximum(big, z.abs()), (freq * count).abs())
        z = z - pres * (count > 0)
        big = torch.maximum(big, z.abs())
        if mask is not None:
            words = (mask if mask.dim() == 1 else mask[b if mask.shape[0] > 1 else 0]).cpu().long() & 0xFFFFFFFF
            v = torch.arange(V)
            z = torch.where((words[v // 32] >> (v % 32)) & 1 == 0, torch.full_like(z, -math.inf), z)
        out[b], top[b] = z, big
    return out, top


def close(got, ref, top):
    got = got.double().cpu()
    assert torch.equal(got == -math.inf, ref == -math.inf) and torch.equal(torch.isnan(got), torch.isnan(ref))
    fine = torch.isfinite(ref)
    tol = 5 * 2.0 ** -24 * top
    return fine, tol, got


def check(got, ref, top, half):
    fine, tol, g = close(got, ref, top)
    if half:
        tol = tol + (ref.abs() * 2.0 ** -11).clamp_min(2.0 ** -25)
    assert bool(((g - ref).abs() <= tol)[fine].all())


def make(seed, B, V, dtype, H, P, per_row, bias, mask, wide=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=DEV)
    x = (r(B, V) * 4).to(dtype)
    history = ints(-1, max(2, V // 3 + 2), B, H).to(wide) if H else None     # many repeats, some ids passed over
    if H:
        history[:, ::3] = history[:, :1].clone()
    lengths = ints(0, H + 2, B).to(wide) if H else None
    prompt = ints(0, V + 1, *((P,) if P % 2 else (B, P))).to(wide) if P else None
    rules = [torch.rand(B, generator=g, device=DEV) + 0.7, r(B) * 0.3, r(B)] if per_row else [1.3, 0.25, 0.5]
    rows = {"none": None, "vector": (), "one": (1,), "row": (B,)}
    b = None if bias == "none" else r(*rows[bias], V)
    m = None if mask == "none" else ints(-2 ** 31, 2 ** 31, *rows[mask], (V + 31) // 32).int()
    return x, history, lengths, prompt, rules, b, m


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,V,H,P,per_row,bias,mask", [
    (1, 1, 1, 0, False, "none", "none"), (1, 151936, 70, 301, False, "none", "none"), (3, 1001, 0, 0, False, "row", "row"),
    (4, 33, 50, 7, True, "vector", "vector"), (2, 2049, 4097, 8, True, "one", "one"), (70, 65535, 20, 0, True, "none", "row"),
    (5, 32003, 1000, 999, False, "vector", "one"), (40, 152064, 600, 64, True, "row", "vector"), (2, 7, 0, 3, False, "none", "none")])
def test_adjust_logits(K, B, V, H, P, per_row, bias, mask, dtype):
    x, history, lengths, prompt, rules, b, m = make(V + B, B, V, dtype, H, P, per_row, bias, mask)
    keep = x.clone()
    kw = dict(lengths=lengths, prompt=prompt, repetition=rules[0], frequency=rules[1], presence=rules[2], bias=b, mask=m)
    got = K.adjust_logits(x, history, **kw)
    assert torch.equal(x, keep)
    ref, top = plain(x, history, lengths, prompt, rules, b, m)
    check(got, ref, top, dtype is torch.float16)
    if history is not None:   # ids of 32 bits; all of the history
        kw.update(lengths=lengths.int(), prompt=None if prompt is None else prompt.int())
        assert torch.equal(K.adjust_logits(x, history.int(), **kw), got)
        kw.update(lengths=None)
        ref, top = plain(x, history, None, prompt, rules, b, m)
        check(K.adjust_logits(x, history, **kw), ref, top, dtype is torch.float16)
    kw.update(lengths=lengths)
    assert K.adjust_logits(x, history, out=x, **kw) is x and torch.equal(x, got)   # in place


def test_adjust_logits_rows(K):
    """Rows inside wider ones, one row of logits for all, a vector, a slice of a token log."""
    wide = torch.randn(6, 5000, device=DEV)
    log = torch.randint(0, 4000, (6, 90), device=DEV)
    x = wide[:, 3:4004]
    ref, top = plain(x, log[:, 2:50], None, None, [1.2, 0.1, 0.2], None, None)
    got = K.adjust_logits(x, log[:, 2:50], repetition=1.2, frequency=0.1, presence=0.2)
    check(got, ref, top, False)
    out = torch.full((6, 5000), 9.0, device=DEV)
    K.adjust_logits(x, log[:, 2:50], repetition=1.2, frequency=0.1, presence=0.2, out=out[:, 500:4501])
    assert torch.equal(out[:, 500:4501], got) and bool((out[:, :500] == 9).all()) and bool((out[:, 4501:] == 9).all())
    one = x[:1].expand(6, 4001)
    ref, top = plain(one, log, None, None, [1.2, 0.0, 0.0], None, None)
    check(K.adjust_logits(one, log, repetition=1.2), ref, top, False)
    v = K.adjust_logits(x[0], log[0], presence=1.0)
    assert v.shape == (4001,) and torch.equal(v, K.adjust_logits(x[:1], log[:1], presence=1.0)[0])


def test_adjust_logits_nothing_to_do(K):
    x = torch.randn(3, 777, device=DEV)
    h = torch.randint(0, 777, (3, 20), device=DEV)
    assert torch.equal(K.adjust_logits(x), x) and torch.equal(K.adjust_logits(x, h), x)
    assert torch.equal(K.adjust_logits(x, h[:, :0], presence=1.0), x)
    assert torch.equal(K.adjust_logits(x, h, torch.full((3,), -5, device=DEV), presence=1.0), x)
    assert K.adjust_logits(x[:0], h[:0]).shape == (0, 777)


def test_adjust_logits_special_values(K):
    """Infinities and NaN keep to their tokens; a mask hides them; a row may be masked whole; the
    lowest value of the type is a value."""
    x = torch.randn(2, 100, device=DEV)
    x[0, 3], x[0, 4], x[0, 5], x[0, 6] = float("nan"), math.inf, -math.inf, torch.finfo(torch.float32).min
    h = torch.tensor([[3, 4, 5, 6, 7], [1, 1, 1, 1, 1]], device=DEV)
    got = K.adjust_logits(x, h, repetition=1.5, frequency=0.5, presence=0.25)
    assert math.isnan(float(got[0, 3])) and float(got[0, 4]) == math.inf and float(got[0, 5]) == -math.inf
    assert float(got[0, 6]) == -math.inf      # 1.5 times the lowest value
    assert int(torch.isnan(got).sum()) == 1 and int(torch.isinf(got).sum()) == 3
    mask = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    mask[0, 0] = ~(1 << 3)
    mask[1] = 0
    got = K.adjust_logits(x, h, mask=mask)
    assert float(got[0, 3]) == -math.inf and bool((got[1] == -math.inf).all()) and torch.equal(got[0, 7:], x[0, 7:])


def test_adjust_logits_long_repeats(K):
    """A token 40000 times in the history: whole counts."""
    x = torch.zeros(1, 50, device=DEV)
    h = torch.full((1, 40001), 11, device=DEV)
    h[0, 77] = 12
    got = K.adjust_logits(x, h, frequency=0.5, presence=1.0)
    want = torch.zeros(1, 50, device=DEV)
    want[0, 11], want[0, 12] = -20001.0, -1.5
    assert torch.equal(got, want)


def test_adjust_logits_graph_stream_two_calls(K):
    """A captured call reads histories and lengths when it is replayed; calls on two streams at once."""
    x, h = torch.randn(4, 30000, device=DEV), torch.randint(0, 30000, (4, 64), device=DEV)
    n = torch.zeros(4, dtype=torch.int64, device=DEV)
    out = torch.empty_like(x)
    K.adjust_logits(x, h, n, repetition=1.1, presence=0.5, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.adjust_logits(x, h, n, repetition=1.1, presence=0.5, out=out)
    for step in range(4):
        n.fill_(16 * step)
        x.normal_()
        graph.replay()
        assert torch.equal(out, K.adjust_logits(x, h, n, repetition=1.1, presence=0.5))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = K.adjust_logits(x, h, repetition=1.3)
    with torch.cuda.stream(s2):
        b = K.adjust_logits(x, h, repetition=1.7)
    torch.cuda.synchronize()
    assert torch.equal(a, K.adjust_logits(x, h, repetition=1.3)) and torch.equal(b, K.adjust_logits(x, h, repetition=1.7))


def test_adjust_logits_refusals(K):
    x, h = torch.randn(2, 64, device=DEV), torch.zeros(2, 5, dtype=torch.int64, device=DEV)
    one = torch.ones(2, device=DEV)
    bad = [dict(repetition=0.0), dict(repetition=float("nan")), dict(presence=math.inf), dict(frequency=one.double()),
           dict(repetition=torch.ones(3, device=DEV)), dict(bias=torch.zeros(63, device=DEV)),
           dict(bias=torch.zeros(2, 64, device=DEV).half()), dict(mask=torch.zeros(1, dtype=torch.int32, device=DEV)),
           dict(mask=torch.zeros(2, 2, device=DEV)), dict(history=h.float()), dict(history=h[:1]), dict(history=h.cpu()),
           dict(history=h, lengths=torch.zeros(3, dtype=torch.int64, device=DEV)), dict(prompt=torch.zeros(3, device=DEV)),
           dict(prompt=torch.zeros(3, 4, dtype=torch.int64, device=DEV)), dict(out=x.half()), dict(out=x[0]),
           dict(history=h.t().contiguous().t())]
    for kw in bad:
        with pytest.raises(ValueError):
            K.adjust_logits(x, **kw)
    for y in (x.double(), x.cpu(), x[:, :0], x[None]):
        with pytest.raises(ValueError):
            K.adjust_logits(y)
    with pytest.raises(RuntimeError):    # rows of the output that share memory
        K.adjust_logits(x, out=torch.empty(1, 64, device=DEV).expand(2, 64))
