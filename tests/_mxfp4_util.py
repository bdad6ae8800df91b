"""Inputs and bounds for the tests of the K/V pool in 4 bits."""
from __future__ import annotations

import torch

from oracle import mxfp4_oracle as mx


def rows(n, n_kv, d, seed, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, n_kv, d, generator=g) * scale).to(dtype)


def pool(num_slots, n_kv, d, seed, dtype=torch.bfloat16):
    """Codes and block bytes of random rows, blocks of very different size among them."""
    g = torch.Generator().manual_seed(seed)
    sizes = torch.exp2(torch.randint(-3, 4, (num_slots, n_kv, d // 32), generator=g).float()).repeat_interleave(32, -1)
    k = (torch.randn(num_slots, n_kv, d, generator=g) * sizes.pow(0.25)).to(dtype)
    v = (torch.randn(num_slots, n_kv, d, generator=g) * sizes).to(dtype)
    return mx.quantised(k, v)


def listed(lens, num_slots, seed):
    """Distinct slots for requests of `lens` keys."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(num_slots, generator=g)[: sum(lens)].to(torch.int32)


def indptr(lens, start=0):
    return torch.cumsum(torch.tensor([start] + list(lens)), 0).to(torch.int32)


def tolerance(spread, score, out, d, dtype=torch.bfloat16, cut=False):
    """How far a result may be off its definition in 64 bits, entry by entry.

    With A = sum_j w_j |v_j|: weights w_j (1 + e_j) in the sum over v and in their own sum give (out + sum w e v) / (1 + sum w e), off by at
    most (A + |out|) max|e| / (1 - max|e|).  They are rounded to the type of q, e up to half a step (2^-8 bf16, 2^-11 half), or cut, e up to a
    whole one.  The result is rounded by half a step of itself.  Scores are sums of d products in 32 bits: off by (d + 2) 2^-24 sum |q k| at most, and a weight, relative to the
    others, by twice that.  exp2, sums of weights and the merge of partials in 32 bits: 2^-18 of A is more than they take.
    """
    half_step = torch.finfo(dtype).eps / 2
    weights = half_step * (2 if cut else 1) * (1 + 2.0 ** -6)
    smallest = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}[dtype]  # half the step of half's smallest numbers, and weights below them
    return weights * (spread + out.abs()) + half_step * out.abs() * (1 + half_step * 4) + spread * (2 * (d + 2) * 2.0 ** -24 * score[..., None] + 2.0 ** -18) + smallest * (1 + spread)


def assert_within(got, out, spread, tol, what=""):
    """`got` of the rows that some request covers (`spread` is a number there)."""
    covered = ~torch.isnan(spread[..., 0]).any(-1) if spread.dim() == 3 else slice(None)
    g, o, t = got.double().cpu()[covered], out[covered], tol[covered]
    assert torch.isfinite(g).all(), f"{what}: not finite"
    over = (g - o).abs() / t.clamp_min(1e-30)
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"
    return worst
