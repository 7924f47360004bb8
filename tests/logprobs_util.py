"""Token log probabilities in float64, and how far fp32 sums may be from them."""

from __future__ import annotations

import torch


def reference(logits: torch.Tensor, tokens: torch.Tensor, scale: float, top: int = 0):
    """(logprobs, entropy, top_logprobs, top_tokens) of 2-D logits and tokens in
    float64 on the CPU."""
    x = logits.detach().cpu().double()
    tokens = tokens.cpu()
    vocab = x.shape[1]
    logp = torch.log_softmax(x * scale, -1)
    picked = logp.gather(1, tokens.clamp(0, vocab - 1))
    picked = picked.masked_fill(tokens < 0, 0.0).masked_fill(tokens >= vocab, float("nan"))
    entropy = torch.special.entr(logp.exp()).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return picked, entropy, logp.gather(1, order), order


def gradient(logits, tokens, scale, grad_logprobs, grad_entropy):
    """The gradient's formula in float64, and the sum of its terms' magnitudes."""
    x = logits.detach().cpu().double()
    tokens = tokens.cpu()
    logp = torch.log_softmax(x * scale, -1)
    p = logp.exp()
    kept = logp.masked_fill(p == 0, 0.0)
    entropy = torch.special.entr(p).sum(-1, keepdim=True)
    g = torch.zeros(tokens.shape, dtype=torch.float64) if grad_logprobs is None else grad_logprobs.cpu().double()
    g = g.masked_fill(tokens < 0, 0.0)
    h = torch.zeros(x.shape[0], 1, dtype=torch.float64) if grad_entropy is None else grad_entropy.cpu().double()[:, None]
    at = tokens.clamp(min=0)
    grad = -p * (g.sum(-1, keepdim=True) + h * (kept + entropy))
    size = p * (g.abs().sum(-1, keepdim=True) + h.abs() * (kept.abs() + entropy))
    return scale * grad.scatter_add(1, at, g), scale * size.scatter_add(1, at, g.abs())


def sum_error(vocab: int) -> float:
    """Relative error of a row's sum: at most vocab / 256 terms one after the
    other in a thread (a chunk has 256), each of a few roundings (its exponent's
    fma is exact to one, v_exp_f32 to one), then about 30 joins."""
    return 2.0**-24 * (vocab / 256 + 64)


def logprob_tolerance(ref: torch.Tensor, vocab: int) -> torch.Tensor:
    """|x - m| * scale and ln(sum) are each at most |logprob| + ln(vocab) and
    rounded a few times."""
    return sum_error(vocab) + 2.0**-22 * (ref.abs() + 12.0)


def entropy_tolerance(ref: torch.Tensor, vocab: int) -> torch.Tensor:
    """H = ln l - t / l: the sums' errors relative to ln l and t / l, each at
    most H + ln(vocab) <= H + 12."""
    return 3 * sum_error(vocab) * (ref.abs() + 12.0)


def close(got: torch.Tensor, ref: torch.Tensor, tolerance: torch.Tensor) -> None:
    """Equal, both NaN, or within the tolerance. Results are fp32 (or narrower): a
    value past fp32's range (two logits at the type's ends, 6.8e38 apart) is an
    infinity there."""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    ref = torch.where(ref.abs() > torch.finfo(torch.float32).max, ref.float().double(), ref)
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~same & ~((got - ref).abs() <= tolerance)
    assert not bad.any(), (got[bad][:5], ref[bad][:5])
