"""8-bit blocks, the projections on them and the embedding in 64 bits, from their definitions.

A block (128 columns of a row, or 128 x 128 of a weight) is e4m3 values with a
scale 2^e, e the least integer with max |finite x| <= 448 2^e, at least -127 and 0
for a block of zeros; what is not finite becomes NaN.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

BLOCK = 128
E4M3_MAX = 448.0


def half_step(v: torch.Tensor) -> torch.Tensor:
    """Half the spacing of e4m3 at |v|: 2^-4 of the power of two below, 2^-10 where e4m3 is subnormal."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    step = 2 * half_step(v)
    return torch.round(v / step) * step  # (ties to even, as torch.round's)


def quantize(x: torch.Tensor, rows: int):
    """(values, scale of each value, scale of each block) of a matrix in blocks of ``rows`` x 128, in 64 bits."""
    x = x.double()
    m, k = x.shape
    full = F.pad(x, (0, -k % BLOCK, 0, -m % rows)).reshape(-(-m // rows), rows, -(-k // BLOCK), BLOCK)
    amax = torch.where(full.isfinite(), full.abs(), torch.zeros_like(full)).amax((1, 3))
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -200) / E4M3_MAX))
    e = torch.where(E4M3_MAX * torch.exp2(e - 1) >= amax, e - 1, e)
    e = torch.where(E4M3_MAX * torch.exp2(e) < amax, e + 1, e).clamp(min=-127)
    scale = torch.exp2(torch.where(amax == 0, torch.zeros_like(e), e))
    each = scale[:, None, :, None].expand(full.shape).reshape(-1, full.shape[2] * BLOCK)[:m, :k]
    q = round_e4m3(x / each)
    return torch.where(x.isfinite(), q, torch.full_like(q, float("nan"))), each, scale


def values(x: torch.Tensor, rows: int) -> torch.Tensor:
    q, each, _ = quantize(x, rows)
    return q * each


def rms_norm(s: torch.Tensor, eps: float):
    """(s / rms(s), 1 / rms(s))"""
    r = (s.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    return s * r, r


def norm_backward(g, ds, y, r):
    """Gradient of s in y = s r(s), the y that was kept, plus the gradient ds that came to s itself."""
    return ds + r * (g - y * (g * y).mean(-1, keepdim=True))


def gate(a, b):
    return a * torch.sigmoid(a) * b


def gate_backward(g, a, b):
    z = torch.sigmoid(a)
    return g * b * z * (1 + a * (1 - z)), g * a * z


def embedding_grad(tokens, dy, vocab, scale, padding_idx=None):
    """(dW, sum of |dy| that entered each of its values)"""
    flat, d = tokens.reshape(-1).long(), dy.shape[-1]
    rows = dy.reshape(-1, d).double()
    ok = (flat >= 0) & (flat < vocab)
    if padding_idx is not None:
        ok &= flat != padding_idx
    dw, size = (torch.zeros(vocab, d, dtype=torch.float64, device=dy.device) for _ in range(2))
    dw.index_add_(0, flat[ok], rows[ok])
    size.index_add_(0, flat[ok], rows[ok].abs())
    return dw * scale, size * abs(scale)
