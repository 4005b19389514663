"""The operators of a batch of continuations of one prompt, as timed cases.

Decoding several continuations of one prompt at once takes, for each step: rotary positions of
the new q and k rows with the write of k and v into every sequence's own cache, attention of every
sequence over the shared prompt's keys and its own, and the rules on the logits (penalties for
repeated tokens, biases, grammar masks) before the tokens are picked. Head layouts and vocabularies
are those of the two model shapes the framework's synthetic models come in (the 0.5B and the 7B
architecture), plus generic ones.

``own`` False: each operator in elementary torch operations, in 32 bits (angles in 64). True: the
framework's kernels.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "pico-engine_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

# query heads, kv heads, head size: the two model shapes, and generic ones (no groups, one kv head,
# groups of four, an odd count)
HEADS = {"0.5b": (14, 2, 64), "7b": (28, 4, 128), "mha": (16, 16, 64), "mqa": (12, 1, 64), "gqa4": (32, 8, 128),
         "odd": (25, 5, 64)}
ROPE_BASE = 1e6
TYPES = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # one sequence's decode step: latency alone
        dict(name="rope_append_1", kind="append", heads="0.5b", batch=1, capacity=64, type="f32", rot=64,
             interleaved=False, scaling="none", far=300),
        # a large batch past the trained context, caches in half precision
        dict(name="rope_append_96_yarn", kind="append", heads="7b", batch=96, capacity=300, type="f16", rot=128,
             interleaved=False, scaling="yarn", far=60000),
        # q and k of a long prompt
        dict(name="rope_prompt_8191", kind="rope", tokens=8191, n=16, dim=64, type="f32", rot=64, interleaved=False,
             scaling="llama3", far=0, heads_first=False),
        # the keys of a cache rotated to other positions, pairs side by side, half of each head
        dict(name="rope_keys_65537_f16", kind="rope", tokens=65537, n=4, dim=128, type="f16", rot=64, interleaved=True,
             scaling="linear", far=1000000, heads_first=True),
        # a few continuations of a chat prompt
        dict(name="attn_4x277", kind="attn", heads="0.5b", batch=4, prefix=277, capacity=64, type="f32"),
        # best of sixteen after a page of text
        dict(name="attn_16x1500", kind="attn", heads="0.5b", batch=16, prefix=1500, capacity=256, type="f32"),
        # a batch of ragged answers to one document
        dict(name="attn_33x8001_7b", kind="attn", heads="7b", batch=33, prefix=8001, capacity=515, type="f32"),
        # few sequences behind the longest context of the benchmarks, half precision
        dict(name="attn_3x32768_f16", kind="attn", heads="0.5b", batch=3, prefix=32768, capacity=100, type="f16"),
        # many sequences behind it, on the 7B shape
        dict(name="attn_64x32768_7b_f16", kind="attn", heads="7b", batch=64, prefix=32768, capacity=1000, type="f16"),
        # one sequence with penalties only
        dict(name="logits_1", kind="logits", batch=1, vocab=151936, history=70, prompt=300, type="f32", per_row=False,
             bias="none", mask="none"),
        # a batch under grammars, with a bias and long ragged histories
        dict(name="logits_24_grammar", kind="logits", batch=24, vocab=152064, history=1537, prompt=4000, type="f32",
             per_row=True, bias="shared", mask="row"),
        # the largest batch, an odd vocabulary, logits in half precision
        dict(name="logits_256_f16", kind="logits", batch=256, vocab=151643, history=600, prompt=0, type="f16",
             per_row=True, bias="none", mask="shared"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "rope", "attn", "attn", "logits", "logits"])
    scaling = rng.choice(["none", "linear", "ntk", "yarn", "llama3"])
    if kind == "append":
        heads = rng.choice(sorted(HEADS))
        dim = HEADS[heads][2]
        return dict(kind=kind, heads=heads, batch=_log(rng, 1, 256), capacity=_log(rng, 8, 400),
                    type=rng.choice(["f32", "f16"]), rot=rng.choice([dim, dim, dim // 2, 20]),
                    interleaved=rng.random() < 0.5, scaling=scaling, far=_log(rng, 16, 1000000))
    if kind == "rope":
        dim = rng.choice([64, 128, 80, 256])
        return dict(kind=kind, tokens=_log(rng, 1, 65536), n=_log(rng, 1, 20), dim=dim, type=rng.choice(["f32", "f16"]),
                    rot=rng.choice([dim, dim, dim // 2, 20]), interleaved=rng.random() < 0.5, scaling=scaling,
                    far=rng.choice([0, _log(rng, 16, 1000000)]), heads_first=rng.random() < 0.5)
    if kind == "attn":
        return dict(kind=kind, heads=rng.choice(sorted(HEADS)), batch=_log(rng, 1, 64), prefix=_log(rng, 1, 32768),
                    capacity=_log(rng, 1, 1000), type=rng.choice(["f32", "f16"]))
    return dict(kind=kind, batch=_log(rng, 1, 256), vocab=_log(rng, 1000, 152064), history=_log(rng, 1, 4096),
                prompt=rng.choice([0, _log(rng, 1, 8192)]), type=rng.choice(["f32", "f16"]), per_row=rng.random() < 0.5,
                bias=rng.choice(["none", "shared", "row"]), mask=rng.choice(["none", "shared", "row"]))


# ---- inputs -------------------------------------------------------------------------------

def _gen(seed, index):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + index)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _freqs(rot, scaling):
    """Radians a position of every pair and the amplitude, as trained and stretched contexts have them."""
    base, factor, trained = ROPE_BASE, 4.0, 32768
    if scaling == "ntk":
        base *= factor ** (rot / (rot - 2))
    f = [base ** (-2 * j / rot) for j in range(rot // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":  # pairs of many turns in the trained context stay, those of few are slowed
        dim = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), rot - 1)
        slow = [min(max((j - lo) / max(hi - lo, 0.001), 0), 1) for j in range(rot // 2)]
        return [x * (1 - s) + x / factor * s for x, s in zip(f, slow)], 0.1 * math.log(factor) + 1
    if scaling == "llama3":  # the same by wavelength, between a quarter of the trained context and all of it
        share = [min(max((trained * x / (2 * math.pi) - 1) / (4 - 1), 0), 1) for x in f]
        f = [x * (s + (1 - s) / factor) for x, s in zip(f, share)]
    return f, 1.0


def prepare(case, seed):
    g = _gen(seed, 0)
    s = dict(case)
    dt = TYPES[case["type"]]
    if case["kind"] in ("append", "rope"):
        f, s["amp"] = _freqs(case["rot"], case["scaling"])
        s["freqs"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if case["kind"] == "append":
        nh, nkv, hd = HEADS[case["heads"]]
        B, cap = case["batch"], case["capacity"]
        # every sequence has decoded some tokens behind a prompt of `far`
        s["positions"] = case["far"] + torch.randint(0, cap, (B,), generator=g, device="cuda")
        s["qkv"] = _randn(g, B, (nh + 2 * nkv) * hd) * 1.5
        s["k"], s["v"] = _randn(g, B, nkv, cap, hd).to(dt), _randn(g, B, nkv, cap, hd).to(dt)
    elif case["kind"] == "rope":
        T, n, hd = case["tokens"], case["n"], case["dim"]
        s["positions"] = torch.arange(T, device="cuda") + int(torch.randint(0, case["far"] + 1, (1,), generator=g, device="cuda"))
        s["x"] = ((_randn(g, n, T, hd) * 1.5).to(dt).transpose(0, 1) if case["heads_first"] else
                  (_randn(g, T, n, hd) * 1.5).to(dt))
    elif case["kind"] == "attn":
        nh, nkv, hd = HEADS[case["heads"]]
        B, P, cap = case["batch"], case["prefix"], case["capacity"]
        s["q"] = _randn(g, B, nh, hd) * 1.5
        s["kp"], s["vp"] = (_randn(g, nkv, P, hd) * 1.5).to(dt), _randn(g, nkv, P, hd).to(dt)
        s["ko"], s["vo"] = (_randn(g, B, nkv, cap, hd) * 1.5).to(dt), _randn(g, B, nkv, cap, hd).to(dt)
        # the position of each sequence's newest token, whose key is in its cache
        s["positions"] = P + torch.randint(0, cap, (B,), generator=g, device="cuda")
    else:
        B, V, H = case["batch"], case["vocab"], case["history"]
        s["logits"] = (_randn(g, B, V) * 3).to(dt)
        # a language's few frequent words and many rare ones
        words = lambda *shape: (V ** torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64)).long() - 1  # noqa: E731
        s["ids"], s["ids_prompt"] = words(B, H), words(case["prompt"]) if case["prompt"] else None
        s["lengths"] = torch.randint(1, H + 1, (B,), generator=g, device="cuda")
        rule = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=g, device="cuda") if case["per_row"] else (lo + hi) / 2  # noqa: E731
        s["repetition"], s["frequency"], s["presence"] = rule(1.0, 1.4), rule(0.0, 0.5), rule(0.0, 0.8)
        rows = lambda how: {"none": None, "shared": 1, "row": B}[how]  # noqa: E731
        nb, nm, W = rows(case["bias"]), rows(case["mask"]), (V + 31) // 32
        s["b"] = None if nb is None else _randn(g, nb, V) * (torch.rand(nb, V, generator=g, device="cuda") < 0.01)
        # a grammar lets few tokens through: words with three bits of four off
        bits = lambda: torch.randint(-2 ** 31, 2 ** 31, (nm, W), generator=g, device="cuda").int()  # noqa: E731
        s["m"] = None if nm is None else bits() & bits()
    return s


# ---- the operators ------------------------------------------------------------------------

def _rotate(x, positions, freqs, amp, interleaved):
    """x (T, n, hd) in 32 bits, rotated by angles made in 64."""
    t = positions.double()[:, None] * freqs
    c, s = (t.cos() * amp).float()[:, None], (t.sin() * amp).float()[:, None]
    r = 2 * freqs.numel()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    y, z = a * c - b * s, a * s + b * c
    turned = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _append(s):
    nh, nkv, hd = HEADS[s["heads"]]
    B = s["batch"]
    qk = s["qkv"][:, :(nh + nkv) * hd].view(B, nh + nkv, hd)
    qk = _rotate(qk, s["positions"], s["freqs"], s["amp"], s["interleaved"])
    rows, slots = torch.arange(B, device="cuda"), s["positions"] - s["far"]
    s["k"][rows, :, slots] = qk[:, nh:].to(s["k"].dtype)
    s["v"][rows, :, slots] = s["qkv"][:, (nh + nkv) * hd:].view(B, nkv, hd).to(s["v"].dtype)
    return qk[:, :nh]


def _attn(s):
    nh, nkv, hd = HEADS[s["heads"]]
    B, P, cap = s["batch"], s["prefix"], s["capacity"]
    G = nh // nkv
    q = s["q"].view(B, nkv, G, hd) * hd ** -0.5
    ap = torch.matmul(q.transpose(0, 1).reshape(nkv, B * G, hd), s["kp"].float().transpose(1, 2))
    ao = torch.matmul(q, s["ko"].float().transpose(2, 3))
    unseen = torch.arange(cap, device="cuda") > (s["positions"] - P)[:, None, None, None]
    ao = ao.masked_fill(unseen, -math.inf)
    a = torch.softmax(torch.cat([ap.view(nkv, B, G, P).transpose(0, 1), ao], -1), -1)
    o = torch.matmul(a[..., :P].transpose(0, 1).reshape(nkv, B * G, P), s["vp"].float())
    o = o.view(nkv, B, G, hd).transpose(0, 1) + torch.matmul(a[..., P:], s["vo"].float())
    return o.reshape(B, nh, hd)


def _bits(words, vocab):
    at = torch.arange(32, device="cuda", dtype=torch.int32)
    return ((words[..., None] >> at) & 1).flatten(-2)[..., :vocab].bool()


def _column(v):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _logits(s):
    B, V, H = s["batch"], s["vocab"], s["history"]
    z = s["logits"].float()
    if s["b"] is not None:
        z = z + s["b"]
    # ids behind a row's length are counted in a column of their own
    ids = s["ids"].masked_fill(torch.arange(H, device="cuda") >= s["lengths"][:, None], V)
    count = torch.zeros(B, V + 1, device="cuda").scatter_add_(1, ids, torch.ones(B, H, device="cuda"))[:, :V]
    seen = count > 0
    if s["ids_prompt"] is not None:
        seen = seen | (torch.zeros(V, device="cuda").index_fill_(0, s["ids_prompt"], 1.0) > 0)
    rep = _column(s["repetition"])
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - _column(s["frequency"]) * count - _column(s["presence"]) * (count > 0)
    if s["m"] is not None:
        z = z.masked_fill(~_bits(s["m"], V), -math.inf)
    return z.to(s["logits"].dtype)


@torch.inference_mode()
def run(s):
    kind = s["kind"]
    if own:
        from pico_hip import kernels as K
    if kind == "append":
        if own:
            q = K.rope_append(s["qkv"], s["positions"], s["freqs"], HEADS[s["heads"]][0], s["k"], s["v"],
                              slot_offset=-s["far"], amp=s["amp"], interleaved=s["interleaved"])
        else:
            q = _append(s)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if kind == "rope":
        if own:
            return K.rope_positions(s["x"], s["positions"], s["freqs"], amp=s["amp"], interleaved=s["interleaved"])
        return _rotate(s["x"].float(), s["positions"], s["freqs"], s["amp"], s["interleaved"]).to(s["x"].dtype)
    if kind == "attn":
        if own:
            return K.shared_prefix_attn(s["q"], s["kp"], s["vp"], s["ko"], s["vo"], s["positions"],
                                        own_offset=1 - s["prefix"], round_fp16=False)
        return _attn(s)
    if own:
        return K.adjust_logits(s["logits"], history=s["ids"], lengths=s["lengths"], prompt=s["ids_prompt"],
                               repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                               bias=s["b"], mask=s["m"])
    return _logits(s)


def work(case):
    e = 2 if case["type"] == "f16" else 4
    if case["kind"] == "append":
        nh, nkv, hd = HEADS[case["heads"]]
        B = case["batch"]
        return {"bytes": B * (4 * (2 * nh + 2 * nkv) * hd + 2 * e * nkv * hd + 8) + 4 * case["rot"],
                "flops": B * (3 * (nh + nkv) + 20) * case["rot"]}
    if case["kind"] == "rope":
        T, n = case["tokens"], case["n"]
        return {"bytes": T * (2 * e * n * case["dim"] + 8) + 4 * case["rot"], "flops": T * (3 * n + 20) * case["rot"]}
    if case["kind"] == "attn":
        nh, nkv, hd = HEADS[case["heads"]]
        B, P, mean = case["batch"], case["prefix"], (case["capacity"] + 1) / 2  # own keys, on average
        return {"bytes": 2 * e * nkv * hd * (P + B * mean) + 8 * B * nh * hd, "flops": 4 * nh * hd * B * (P + mean)}
    B, V = case["batch"], case["vocab"]
    extra = {"none": 0, "shared": 1, "row": B}
    return {"bytes": 2 * e * B * V + 4 * V * extra[case["bias"]] + V / 8 * extra[case["mask"]] +
            8 * (B * (case["history"] + 1) / 2 + case["prompt"]), "flops": 6 * B * V}


# ---- from the definitions, in 64 bits -----------------------------------------------------

def _turned(x, positions, freqs, amp, interleaved):
    """Every pair as a complex number, times amp e^(i position frequency)."""
    x, r = x.double(), 2 * freqs.numel()
    pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if interleaved else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    w = torch.polar(torch.full((), amp, dtype=torch.float64, device="cuda"), torch.outer(positions.double(), freqs))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w[:, None])
    out = x.clone()
    out[..., :r] = (z if interleaved else z.transpose(-1, -2)).flatten(-2)
    return out


@torch.inference_mode()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _turned(s["x"], s["positions"], s["freqs"], s["amp"], s["interleaved"])
    if case["kind"] == "append":
        nh, nkv, hd = HEADS[case["heads"]]
        rows = s["qkv"].double().unflatten(1, (nh + 2 * nkv, hd))
        turned = _turned(rows[:, :nh + nkv], s["positions"], s["freqs"], s["amp"], s["interleaved"])
        k, v = s["k"].double(), s["v"].double()
        for b, p in enumerate(s["positions"].tolist()):
            k[b, :, p - case["far"]] = turned[b, nh:]
            v[b, :, p - case["far"]] = rows[b, nh + nkv:]
        return {"q": turned[:, :nh], "k": k, "v": v}
    if case["kind"] == "attn":
        nh, nkv, hd = HEADS[case["heads"]]
        out = torch.empty(case["batch"], nh, hd, dtype=torch.float64, device="cuda")
        q = s["q"].double().unflatten(1, (nkv, nh // nkv))
        for b, p in enumerate(s["positions"].tolist()):
            n = p - case["prefix"] + 1
            for j in range(nkv):
                keys = torch.cat([s["kp"][j], s["ko"][b, j, :n]]).double()
                values = torch.cat([s["vp"][j], s["vo"][b, j, :n]]).double()
                scores = q[b, j] @ keys.T / math.sqrt(hd)
                e = torch.exp(scores - scores.amax(1, keepdim=True))
                out[b].unflatten(0, (nkv, nh // nkv))[j] = e @ values / e.sum(1, keepdim=True)
        return out
    V = case["vocab"]
    value = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else v  # noqa: E731
    prompt = torch.zeros(V, dtype=torch.bool, device="cuda")
    if s["ids_prompt"] is not None:
        prompt[s["ids_prompt"]] = True
    out = torch.empty(case["batch"], V, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        z = s["logits"][b].double()
        if s["b"] is not None:
            z = z + s["b"][b if case["bias"] == "row" else 0].double()
        count = torch.bincount(s["ids"][b, :n], minlength=V).double()
        rep = value(s["repetition"], b)
        scale = torch.where(z > 0, torch.full_like(z, 1 / rep), torch.full_like(z, rep))
        z = torch.where((count > 0) | prompt, z * scale, z)
        z = z - value(s["frequency"], b) * count - value(s["presence"], b) * (count > 0).double()
        if s["m"] is not None:
            words = s["m"][b if case["mask"] == "row" else 0]
            v = torch.arange(V, device="cuda")
            z[(words.long()[v // 32] >> (v % 32)) & 1 == 0] = -math.inf
        out[b] = z
    return out
