"""Several continuations of one prompt: decode_shared against the model's own single-sequence decode, and
generate_many against a host loop with the same rules."""

import math

import pytest
import torch

from pico_hip import synth

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def eng(tiny_model):
    from pico_hip.engine import Engine
    return Engine(tiny_model, device="cuda:0")


@pytest.fixture(scope="module")
def eng128(model_dir):
    """A model with heads of 128, one kv head for three query heads."""
    from pico_hip.engine import Engine
    path = model_dir / "tiny-2l-hd128.gguf"
    if not path.exists():
        synth.build(path, synth.tiny_arch(n_layers=2, hidden=256, n_head=3, n_kv=1, head_dim=128, ffn=512, vocab=1024), seed=9)
    return Engine(path, device="cuda:0")


def single(eng, ids, forced):
    """Logits after the prompt and after each forced token, one sequence."""
    cache = eng._empty_cache(len(ids) + len(forced) + 1)
    out = [eng.model.forward(torch.tensor(ids, device=DEV), torch.arange(len(ids), device=DEV), cache)]
    for i, t in enumerate(forced):
        out.append(eng.model.forward(torch.tensor([t], device=DEV), torch.tensor([len(ids) + i], device=DEV), cache))
    return torch.stack(out)


@pytest.mark.parametrize("P,B,dtype", [(5, 1, torch.float32), (33, 3, torch.float32), (33, 3, torch.float16), (700, 40, torch.float32),
                                       (1, 2, torch.float32), (1500, 34, torch.float16)])
@pytest.mark.parametrize("which", ["eng", "eng128"])
def test_decode_shared_matches_single_sequences(which, P, B, dtype, request):
    """Every sequence's logits within 1e-3 of its own decode (the models' criterion; 3e-3 with the keys
    and values rounded to fp16), sequences of different lengths, one of them taking no part."""
    eng = request.getfixturevalue(which)
    m, c = eng.model, eng.cfg
    g = torch.Generator().manual_seed(P)
    ids = torch.randint(0, 1024, (P,), generator=g).tolist()
    steps = 4
    forced = torch.randint(0, 1024, (B, steps), generator=g)
    prefix = eng._empty_cache(P)
    m.forward(torch.tensor(ids, device=DEV), torch.arange(P, device=DEV), prefix)
    prefix = [(k.to(dtype), v.to(dtype)) for k, v in prefix]
    own = [tuple(torch.full((B, c.n_kv_head, steps + 3, c.head_dim), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
           for _ in range(c.n_layers)]
    got = []
    for t in range(steps):
        pos = torch.full((B,), P + t, dtype=torch.int64, device=DEV)
        if B > 2:
            pos[1] = -1
        got.append(m.decode_shared(forced[:, t].to(DEV), pos, prefix, own))
    tol = 1e-3 if dtype is torch.float32 else 3e-3
    for b in [i for i in range(B) if B <= 2 or i != 1][:5] + [B - 1]:
        want = single(eng, ids, forced[b].tolist())[1:]
        for t in range(steps):
            err = float((got[t][b] - want[t]).abs().max() / want[t].abs().max())
            assert err < tol, (b, t, err)
    if B > 2:
        assert all(bool(torch.isnan(x[1]).all()) for kv in own for x in kv)      # nothing written
    assert all(bool(torch.isnan(x[0, :, steps:]).all()) for kv in own for x in kv)


def host_loop(eng, ids, max_tokens, rules, bias, banned):
    """Greedy decoding of one sequence with the rules on the host: (tokens, margin of each pick)."""
    cache = eng._empty_cache(len(ids) + max_tokens)
    logits = eng.model.forward(torch.tensor(ids, device=DEV), torch.arange(len(ids), device=DEV), cache)
    out, margins = [], []
    for t in range(max_tokens):
        z = logits.double().cpu() + bias.double()
        for v in set(ids) | set(out):
            z[v] = z[v] / rules["repetition"] if z[v] > 0 else z[v] * rules["repetition"]
        for v in set(out):
            z[v] -= out.count(v) * rules["frequency"] + rules["presence"]
        z[banned] = -math.inf
        top = z.topk(2)
        margins.append(float(top.values[0] - top.values[1]) / float(logits.abs().max()))
        out.append(int(top.indices[0]))
        logits = eng.model.forward(torch.tensor([out[-1]], device=DEV), torch.tensor([len(ids) + t], device=DEV), cache)
    return out, margins


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("P", [7, 40])
def test_generate_many_greedy_follows_the_rules(eng, P, use_graph):
    g = torch.Generator().manual_seed(3 + P)
    ids = torch.randint(0, 1024, (P,), generator=g).tolist()
    bias = torch.randn(1024, generator=g) * 0.3
    banned = torch.arange(0, 1024, 3)
    words = torch.zeros(32, dtype=torch.int64)
    for v in range(1024):
        if v % 3:
            words[v // 32] |= 1 << (v % 32)
    mask = torch.where(words >= 1 << 31, words - (1 << 32), words).int().to(DEV)
    rules = dict(repetition=1.3, frequency=0.2, presence=0.4)
    want, margins = host_loop(eng, ids, 20, rules, bias, banned)
    got = eng.generate_many(ids, 3, 20, temperature=0.0, bias=bias.to(DEV), mask=mask, eos_id=-2, use_graph=use_graph, **rules)
    assert got[0] == got[1] == got[2] and len(got[0]) == 20
    sure = next((i for i, m in enumerate(margins) if m < 2e-3), 20)     # both sides within 1e-3 of the logits
    assert sure >= 3 and got[0][:sure] == want[:sure]
    assert all(v % 3 for v in got[0])


def test_generate_many_plain_greedy_is_generate(eng):
    ids = [5, 77, 901, 3, 12, 640]
    want, margins = host_loop(eng, ids, 24, dict(repetition=1.0, frequency=0.0, presence=0.0), torch.zeros(1024), [])
    sure = next((i for i, m in enumerate(margins) if m < 2e-3), 24)
    for dtype in (torch.float32, torch.float16):
        got = eng.generate_many(ids, 2, 24, temperature=0.0, eos_id=-2, cache_dtype=dtype)
        assert got[0] == got[1] and got[0][:min(sure, 24)] == want[:sure] or dtype is torch.float16


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-3), (torch.float16, 3e-3)])
def test_generate_many_plain_greedy_with_either_cache(eng, dtype, bound):
    """Without rules the tokens are the host loop's up to the first pick that both sides' bound on the logits leaves
    open, twice that of test_decode_shared_matches_single_sequences."""
    for ids in ([5, 77, 901, 3, 12, 640], list(range(300, 340))):
        want, margins = host_loop(eng, ids, 24, dict(repetition=1.0, frequency=0.0, presence=0.0), torch.zeros(1024), [])
        sure = next((i for i, m in enumerate(margins) if m < 2 * bound), 24)
        got = eng.generate_many(ids, 3, 24, temperature=0.0, eos_id=-2, cache_dtype=dtype)
        assert got[0] == got[1] == got[2] and len(got[0]) == 24
        assert sure >= 3 and got[0][:sure] == want[:sure], (sure, got[0], want)


def test_generate_many_stops_and_samples(eng):
    """A stop token ends its sequence only; sampled continuations differ and repeat with the generator."""
    ids = list(range(20, 40))
    first = eng.generate_many(ids, 8, 40, temperature=1.0, eos_id=-2, generator=torch.Generator(DEV).manual_seed(1))
    again = eng.generate_many(ids, 8, 40, temperature=1.0, eos_id=-2, generator=torch.Generator(DEV).manual_seed(1))
    assert first == again and len({tuple(r) for r in first}) > 1 and all(len(r) == 40 for r in first)
    stop = first[0][5]
    cut = eng.generate_many(ids, 8, 40, temperature=1.0, eos_id=stop, generator=torch.Generator(DEV).manual_seed(1))
    assert cut[0] == first[0][:first[0].index(stop)] and stop not in sum(cut, [])
    assert eng.generate_many([], 2, 5) == [[], []] and eng.generate_many(ids, 0, 5) == []
    assert [len(r) for r in eng.generate_many(ids, 2, 1, temperature=0.0, eos_id=-2)] == [1, 1]
    with pytest.raises(ValueError):
        eng.generate_many(ids, 2, eng.cfg.context_len)
    with pytest.raises(ValueError):
        eng.generate_many(ids, 2, 4, cache_dtype=torch.bfloat16)


@pytest.mark.parametrize("n", [2, 9, 70])
@pytest.mark.parametrize("which", ["eng", "eng128"])
def test_generate_many_graph_is_eager(which, n, request):
    """The captured step replayed with the host's work between gives the eager steps' tokens."""
    eng = request.getfixturevalue(which)
    kw = dict(temperature=0.8, top_k=20, repetition=1.2, frequency=0.1, eos_id=-2)
    ids = list(range(7, 60))
    runs = [eng.generate_many(ids, n, 20, use_graph=g, generator=torch.Generator(DEV).manual_seed(n), **kw) for g in (False, True, True)]
    assert runs[0] == runs[1] == runs[2] and len({tuple(r) for r in runs[0]}) == n


def test_generate_many_refuses_masks_that_leave_nothing(eng):
    mask = torch.full((2, 32), -1, dtype=torch.int32, device=DEV)
    mask[1] = 0
    bias = torch.full((1024,), -math.inf, device=DEV)
    for rules in (dict(mask=mask), dict(bias=bias)):
        with pytest.raises(ValueError):
            eng.generate_many([3, 4, 5], 2, 4, temperature=1.0, eos_id=-2, **rules)
    mask[1, 3] = 1 << 9             # one token is left
    got = eng.generate_many([3, 4, 5], 2, 4, temperature=1.0, eos_id=-2, mask=mask)
    assert got[1] == [3 * 32 + 9] * 4 and len(got[0]) == 4


def test_generate_many_stop_token_that_never_comes(eng):
    """An id that no token has, -1 among them, stops nothing."""
    n = eng.greedy_chunk + 5
    want = eng.generate_many([3, 4, 5], 2, n, temperature=0.0, eos_id=-2)
    assert [len(r) for r in want] == [n, n]
    assert eng.generate_many([3, 4, 5], 2, n, temperature=0.0, eos_id=-1) == want


def test_sample_rows_does_not_wait_for_the_gpu():
    from pico_hip.sampler import sample_rows
    z = torch.randn(4, 300, device=DEV)
    z[3] = -math.inf
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        picks = [sample_rows(z, **kw) for kw in (dict(temperature=0.0), dict(temperature=0.7), dict(temperature=0.7, top_k=5),
                                                 dict(temperature=0.7, top_p=0.9))]
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    assert all(0 <= v < 300 for p in picks for v in p.tolist()) and all(int(p[3]) == 0 for p in picks)


def test_sample_rows_draws_by_the_probabilities():
    """20000 draws of 5 tokens: every count within 5 standard deviations, sqrt(n p (1 - p)), of n p."""
    from pico_hip.sampler import sample_rows
    p, n = torch.tensor([0.5, 0.25, 0.15, 0.1, 0.0]), 20000
    picks = sample_rows(p.log().to(DEV).expand(n, 5), generator=torch.Generator(DEV).manual_seed(5))
    counts = torch.bincount(picks.cpu(), minlength=5).double()
    assert int(counts[4]) == 0 and bool(((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all())


def test_sample_rows_matches_sample():
    from pico_hip.sampler import sample, sample_rows
    z = torch.randn(6, 500, device=DEV) * 3
    z[2, 10:] = -math.inf
    assert sample_rows(z, 0.0).tolist() == [sample(r, 0.0) for r in z]
    for kw in (dict(temperature=0.8), dict(temperature=0.5, top_k=3), dict(temperature=1.0, top_p=0.5), dict(temperature=1.0, top_k=40, top_p=0.9)):
        picks = torch.stack([sample_rows(z, generator=torch.Generator(DEV).manual_seed(i), **kw) for i in range(200)])
        for b in range(6):
            probs = torch.softmax(z[b] / kw["temperature"], -1)
            order = probs.argsort(descending=True)
            allowed = set(order[:kw.get("top_k") or 500].tolist())
            if "top_k" in kw:
                probs = torch.where(probs >= probs[order[kw["top_k"] - 1]], probs, torch.zeros_like(probs))
                probs = probs / probs.sum()
            if "top_p" in kw:
                before = probs[order].cumsum(0) - probs[order]
                allowed &= set(order[before <= kw["top_p"] + 1e-6].tolist())
            assert set(picks[:, b].tolist()) <= allowed
