"""Token sampling over logits (the reference's sampler.py surface, sampler.py:8-27).

Greedy (temperature <= 0) is ``argmax`` (first maximum on ties) followed by one device-to-host
read; otherwise temperature scaling, optional top-k and top-p filtering and a multinomial
draw, all as torch ops on the logits' device.
"""

from __future__ import annotations

import torch


def sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           generator: torch.Generator | None = None) -> int:
    """Draw one token id from 1-D raw ``logits``."""
    if temperature <= 0:
        return int(torch.argmax(logits).item())
    z = logits.float() / temperature
    if top_k > 0:
        kth = torch.topk(z, min(top_k, z.numel())).values[-1]
        z = torch.where(z < kth, torch.full_like(z, float("-inf")), z)
    if top_p < 1.0:
        order = torch.argsort(z, descending=True)
        probs = torch.softmax(z[order], dim=-1)
        cut = torch.cumsum(probs, dim=-1) > top_p
        cut = torch.cat([cut.new_zeros(1), cut[:-1]])  # keep the token that crosses top_p
        z = z.clone()
        z[order[cut]] = float("-inf")
    probs = torch.softmax(z, dim=-1)
    return int(torch.multinomial(probs, 1, generator=generator).item())


def sample_rows(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                generator: torch.Generator | None = None) -> torch.Tensor:
    """``sample`` of every row of (B, V) raw ``logits``: (B,) int64 ids on the logits' device, with no
    read back to the host. A row may hold -inf (tokens that are ruled out); one that holds nothing else
    gives id 0. The draw is a race of exponential times, of which token v's ends first with
    probability p_v (torch.multinomial reads its probabilities back to check them)."""
    if temperature <= 0:
        return torch.argmax(logits, dim=-1)
    z = logits.float() / temperature
    if top_k > 0:
        kth = torch.topk(z, min(top_k, z.shape[-1]), dim=-1).values[:, -1:]
        z = z.masked_fill(z < kth, float("-inf"))
    if top_p < 1.0:
        order = torch.argsort(z, dim=-1, descending=True)
        probs = torch.softmax(z.gather(-1, order), dim=-1)
        cut = torch.cumsum(probs, dim=-1) > top_p
        cut = torch.cat([torch.zeros_like(cut[:, :1]), cut[:, :-1]], dim=-1)  # keep the token that crosses top_p
        z = z.masked_fill(torch.zeros_like(cut).scatter(-1, order, cut), float("-inf"))
    probs = torch.softmax(z, dim=-1)
    times = torch.empty_like(probs).exponential_(generator=generator).clamp_(min=torch.finfo(probs.dtype).tiny)
    return torch.argmax(probs / times, dim=-1)
