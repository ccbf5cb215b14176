"""Embedding lookup with a scale, its gradient by sorted tokens, on gfx950.

The lookups of KernelDev's ``GPTModel`` (``model.py:127-178``).  The gradient
adds the rows of equal tokens in fp32 in the order of their positions, without
atomics: the same inputs give the same bits.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

torch.library.define("kdattn::embed", "(Tensor tokens, Tensor weight, float scale) -> Tensor")
torch.library.define("kdattn::embed_grad",
                     "(Tensor tokens, Tensor dy, SymInt vocab, float scale, int padding_idx) -> Tensor")


@torch.library.register_fake("kdattn::embed")
def _(tokens, weight, scale):
    _lib.native()
    return weight.new_empty((*tokens.shape, weight.shape[1]))


@torch.library.register_fake("kdattn::embed_grad")
def _(tokens, dy, vocab, scale, padding_idx):
    return dy.new_empty((vocab, dy.shape[-1]))


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return torch.ops.kdattn.embed(tokens, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return None, torch.ops.kdattn.embed_grad(tokens, dy, ctx.vocab, ctx.scale, ctx.padding_idx), None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[tokens]`` ``[..., D]``, differentiable once in ``weight`` ``[V, D]`` (bf16, fp16 or fp32).

    ``tokens`` are int64 or int32 of any shape on the weight's GPU.  A token outside ``0 .. V - 1`` reads nothing: its
    row is NaN, and it takes no part in the gradient.  ``padding_idx`` (negative: from the end) names a token whose row of the
    gradient stays zero; it is looked up like any other."""
    if _lib.eager(tokens, weight) and (y := _lib.native().embedding(tokens, weight, scale, padding_idx)) is not None:
        return y
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [V, D], got {tuple(weight.shape)}")
    if weight.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"weight must be bf16, fp16 or fp32, got {weight.dtype}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32, got {tokens.dtype}")
    pad = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx must be within the vocabulary of {weight.shape[0]}, got {padding_idx}")
        pad = int(padding_idx) % weight.shape[0]
    if weight.device.type != "cuda" or tokens.device != weight.device:
        raise ValueError("tokens and weight must be on the same GPU (no CPU fallback)")
    if not torch.compiler.is_compiling():
        _lib.native()
    return _Embedding.apply(tokens, weight, float(scale), pad)


__all__ = ["embedding"]
