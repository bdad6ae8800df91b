"""The K/V pool in 4 bits, in 64 bits on the CPU: what its writers leave, what it stands for, and attention over it.

Codes are 4-bit floats (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign, dim 2i in the low half of byte i), a block of 32 dims has one byte b for the
factor 2^(b - 127): the smallest with which no value lies beyond 6, b in [2, 252].  A head whose row of K or V is not finite leaves
255 in K's block bytes and zero codes.  The reference has no such pool.
"""
from __future__ import annotations

import torch

BLOCK = 32
CODES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# halfway between neighbouring codes, and whether the one above is the even one
BORDERS = (CODES[1:] + CODES[:-1]) / 2
EVEN_ABOVE = torch.tensor([False, True] * 3 + [False])


def block_bytes(x: torch.Tensor) -> torch.Tensor:
    """``(..., d)`` finite values -> ``(..., d / 32)`` block bytes."""
    amax = x.double().unflatten(-1, (-1, BLOCK)).abs().amax(-1)
    mantissa, exponent = torch.frexp(amax / 6)  # mantissa in [0.5, 1): 2^exponent, but 2^(exponent - 1) for 0.5 itself
    return (127 + exponent - (mantissa == 0.5).to(exponent.dtype)).clamp(2, 252).masked_fill(amax == 0, 2)


def quantised(k: torch.Tensor, v: torch.Tensor):
    """Rows ``(n, heads, d)`` -> codes ``(n, heads, 2, d / 2)`` and block bytes ``(n, heads, 2, d / 32)``, uint8."""
    x = torch.stack((k.double(), v.double()), 2)
    fine = torch.isfinite(x).all(-1).all(-1)
    x = torch.where(fine[:, :, None, None], x, torch.zeros_like(x))
    byte = block_bytes(x)
    size = torch.ldexp(x.abs().unflatten(-1, (-1, BLOCK)), (127 - byte)[..., None])
    code = torch.zeros(size.shape, dtype=torch.int64)
    for border, even_above in zip(BORDERS.tolist(), EVEN_ABOVE.tolist()):
        code += (size >= border) if even_above else (size > border)
    code = (code + 8 * torch.signbit(x).unflatten(-1, (-1, BLOCK))).flatten(-2)
    byte[:, :, 0] = torch.where(fine[:, :, None], byte[:, :, 0], torch.full_like(byte[:, :, 0], 255))
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), byte.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes ``(..., d / 2)`` under block bytes ``(..., d / 32)`` stand for: ``(..., d)`` float64."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    x = CODES[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
    factor = torch.ldexp(torch.ones((), dtype=torch.float64), scales.long() - 127).masked_fill(scales == 255, float("nan"))
    return (x.unflatten(-1, (-1, BLOCK)) * factor[..., None]).flatten(-2)


def norm_rope(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor, eps: float, base: float) -> torch.Tensor:
    x, half = x.double(), x.shape[-1] // 2
    y = weight.double() * x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    angle = positions.double()[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = y[..., :half], y[..., half:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def attention(q, codes, scales, qo_indptr, kv_indptr, kv_indices, prefix_lens, sm_scale, *, max_len_extend=None,
              is_cross=False, window=0):
    """``(out, spread, score)`` in float64 for the rows of ``q``; None for ``qo_indptr`` and ``prefix_lens`` means decode.

    ``spread[r, h, d] = sum_j w_j |v_jd|`` and ``score[r, h] = sm_scale max_j sum_d |q_d k_jd|`` are what rounding errors
    are relative to.  Rows that no request covers are NaN in ``spread``.
    """
    n, n_q, d = q.shape
    n_kv = codes.shape[1]
    if qo_indptr is None:
        qo = list(range(n + 1))
    else:
        qo = qo_indptr.tolist()
    kv = kv_indptr.tolist()
    out, spread = torch.zeros(n, n_q, d, dtype=torch.float64), torch.full((n, n_q, d), float("nan"), dtype=torch.float64)
    score = torch.zeros(n, n_q, dtype=torch.float64)
    for b in range(len(kv) - 1):
        slots = kv_indices[kv[b]:kv[b + 1]].long()
        x = values(codes[slots], scales[slots])  # (keys, heads, 2, d)
        rows = qo[b + 1] - qo[b]
        if max_len_extend is not None:
            rows = min(rows, max_len_extend)
        prefix = len(slots) - 1 if prefix_lens is None else int(prefix_lens[b])
        for i in range(rows):
            pos = prefix + i
            seen = torch.ones(len(slots), dtype=torch.bool)
            j = torch.arange(len(slots))
            if not is_cross:
                seen &= j <= pos
            if window > 0:
                seen &= j >= pos - window + 1
            r = qo[b] + i
            spread[r] = 0
            if not bool(seen.any()):
                continue
            k, v = x[seen][:, :, 0], x[seen][:, :, 1]
            qr = q[r].double().view(n_kv, n_q // n_kv, d)
            s = torch.einsum("hgd,jhd->hgj", qr, k) * sm_scale
            score[r] = (torch.einsum("hgd,jhd->hgj", qr.abs(), k.abs()).amax(-1) * sm_scale).reshape(-1)
            w = torch.softmax(s, -1)
            out[r] = torch.einsum("hgj,jhd->hgd", w, v).reshape(n_q, d)
            spread[r] = torch.einsum("hgj,jhd->hgd", w, v.abs()).reshape(n_q, d)
    return out, spread, score
