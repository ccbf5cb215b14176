"""The transformer block's projections in 8 bits on gfx950.

An 8-bit block is 128 consecutive columns of a row (128 x 128 values of a
weight) held as OCP e4m3 with one power-of-two scale ``2^e``: ``e`` is the least
integer with ``max |x| <= 448 * 2^e`` over the block's finite values (0 for a
block of zeros), kept as ``float8_e8m0fnu``.  The matrix instruction applies such
scales by itself, and multiplying by them is exact, so the one rounding is the
one to e4m3 (to nearest, ties to even).  Values that are not finite become NaN
and leave the rest of their block as it is.

* :func:`quantize_rows`, :func:`quantize_weight`, :func:`dequantize` -- to and from blocks;
* :func:`fp8_matmul` -- the product of blocks;
* :func:`add_rms_norm_fp8` -- the residual's addition, RMSNorm (``model.py:31-39``) and the rounding in one pass;
* :func:`norm_projection`, :func:`fp8_projection`, :func:`swiglu_projection` -- differentiable: these
  projections (``model.py:42-96``) with their products in 8 bits, which keep their
  activations for the backward in 8 bits only.

Backward of the three: the gradient of the operand is the 8-bit product of the
incoming gradient, rounded to blocks along its columns, with the forward's 8-bit
weight; the weight's gradient is the 16-bit gradient times the kept 8-bit operand
(straight through the rounding, as the fp8 attention scores are), in fp32 sums
rounded once.  RMSNorm's and the gate's gradients are formed from what was kept.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

BLOCK = 128
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class BlockFp8(NamedTuple):
    """Values ``data`` (float8_e4m3fn) and their ``scale`` (float8_e8m0fnu): a block stands for data * scale."""

    data: torch.Tensor
    scale: torch.Tensor


# ------------------------------------------------- operators (csrc/kd_torch_block8.cpp)
_SCHEMAS = {
    "quant_rows8": "(Tensor[] x) -> (Tensor, Tensor)",
    "quant_weight8": "(Tensor[] w, bool transpose) -> (Tensor, Tensor, Tensor, Tensor)",
    "matmul8": "(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, ScalarType dtype, bool fast=False) -> Tensor",
    "norm8": "(Tensor x, Tensor? delta, float eps) -> (Tensor, Tensor, Tensor, Tensor)",
    "norm8_bwd": "(Tensor g, Tensor? ds, Tensor y, Tensor scale, Tensor rstd, ScalarType dtype) -> Tensor",
    "gate8": "(Tensor a, Tensor b, bool keep) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
    "gate8_bwd": "(Tensor dy, Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, ScalarType dtype) -> (Tensor, Tensor)",
    "weight_grad8": "(Tensor[] dy, Tensor x, Tensor x_scale, int K) -> Tensor",
}
for _name, _schema in _SCHEMAS.items():
    torch.library.define(f"kdattn::{_name}", _schema)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _bytes8(like, rows, cols):
    return like.new_empty((rows, (cols + 15) // 16 * 16), dtype=_E4M3)


def _scales(like, rows, nb):
    return like.new_empty((rows, nb), dtype=_E8M0)


def _fake(name):
    def put(f):
        def with_library(*args):
            _lib.native()  # (a traced program runs the kernels later: they are there from now on)
            return f(*args)

        torch.library.register_fake(f"kdattn::{name}")(with_library)
        return f

    return put


@_fake("quant_rows8")
def _(xs):
    x, total = xs[0], sum(t.shape[1] for t in xs)
    return _bytes8(x, x.shape[0], total), _scales(x, x.shape[0], _blocks(total))


@_fake("quant_weight8")
def _(ws, transpose):
    w, n, k = ws[0], sum(t.shape[0] for t in ws), ws[0].shape[1]
    y, s = _bytes8(w, n, k), _scales(w, _blocks(n), _blocks(k))
    return (y, s, _bytes8(w, k, n), _scales(w, _blocks(k), _blocks(n))) if transpose else (
        y, s, _bytes8(w, 0, 0), _scales(w, 0, 0))


@_fake("matmul8")
def _(a, a_scale, b, b_scale, dtype, fast=False):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=dtype)


@_fake("norm8")
def _(x, delta, eps):
    rows, d = x.shape
    return (x.new_empty((0,)) if delta is None else torch.empty_like(x, memory_format=torch.contiguous_format),
            _bytes8(x, rows, d), _scales(x, rows, _blocks(d)), x.new_empty((rows,), dtype=torch.float32))


@_fake("norm8_bwd")
def _(g, ds, y, scale, rstd, dtype):
    return g.new_empty(g.shape, dtype=dtype)


@_fake("gate8")
def _(a, b, keep):
    rows, h = a.shape
    kept = rows if keep else 0
    return (_bytes8(a, rows, h), _scales(a, rows, _blocks(h)), _bytes8(a, kept, h), _scales(a, kept, _blocks(h)),
            _bytes8(a, kept, h), _scales(a, kept, _blocks(h)))


@_fake("gate8_bwd")
def _(dy, a, a_scale, b, b_scale, dtype):
    return dy.new_empty(dy.shape, dtype=dtype), dy.new_empty(dy.shape, dtype=dtype)


@_fake("weight_grad8")
def _(dys, x, x_scale, K):
    return dys[0].new_empty((sum(d.shape[1] for d in dys), K))


def _ops():
    if not torch.compiler.is_compiling():
        _lib.native()
    return torch.ops.kdattn


# ----------------------------------------------------------------- blocks
_HALF = (torch.bfloat16, torch.float16)


def _check_operand(name, x, types=_HALF, of=8):
    if x.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")
    if x.dtype not in types:
        raise ValueError(f"{name} must be {' or '.join(str(t)[6:] for t in types)}, got {x.dtype}")
    if x.shape[-1] < of or x.shape[-1] % of:
        raise ValueError(f"{name}'s last dimension must be a multiple of {of}, got {x.shape[-1]}")


def _check_gpu(name, *xs):
    if xs[0].device.type != "cuda" or any(x.device != xs[0].device for x in xs):
        raise ValueError(f"{name} must be on one GPU (no CPU fallback)")


def quantize_rows(x: torch.Tensor) -> BlockFp8:
    """``x`` ``[..., K]`` (bf16, fp16 or fp32; K a multiple of 16) in blocks of 128 columns of a row:
    data ``[..., K]`` and scale ``[..., ceil(K / 128)]``.  Not differentiable."""
    if _lib.eager(x) and (got := _lib.native().quantize_rows(x)) is not None:
        return BlockFp8(*got)
    _check_operand("x", x, (*_HALF, torch.float32), 16)
    _check_gpu("x", x)
    data, scale = _ops().quant_rows8([x.detach().reshape(-1, x.shape[-1])])
    return BlockFp8(data.view(x.shape), scale.view(*x.shape[:-1], _blocks(x.shape[-1])))


def quantize_weight(w: torch.Tensor) -> BlockFp8:
    """``w`` ``[N, K]`` (bf16, fp16 or fp32; K a multiple of 16) in blocks of 128 x 128: data ``[N, K]`` and
    scale ``[ceil(N / 128), ceil(K / 128)]``.  Not differentiable."""
    _check_operand("w", w, (*_HALF, torch.float32), 16)
    if w.dim() != 2 or w.shape[0] < 1:
        raise ValueError(f"w must be [N, K], got {tuple(w.shape)}")
    _check_gpu("w", w)
    return BlockFp8(*_ops().quant_weight8([w.detach()], False)[:2])


def _check_blocks(name, x, two_dim=False):
    if x.data.dtype != _E4M3 or x.scale.dtype != _E8M0:
        raise ValueError(f"{name} must be float8_e4m3fn values with float8_e8m0fnu scales, got {x.data.dtype} and "
                         f"{x.scale.dtype}")
    if x.data.dim() < 1 or (two_dim and x.data.dim() != 2) or x.data.shape[-1] < 16 or x.data.shape[-1] % 16:
        raise ValueError(f"{name} must be {'[N, K]' if two_dim else '[..., K]'}, K a multiple of 16, got "
                         f"{tuple(x.data.shape)}")


def dequantize(x: BlockFp8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that blocks of rows or of a weight stand for (``data * scale``), in torch operations.

    Rows have a scale row each; a weight has one for each 128 of its rows."""
    x = BlockFp8(*x)
    k, rows = x.data.shape[-1], x.data.shape[:-1]
    scale = x.scale.float()
    if tuple(x.scale.shape[:-1]) != tuple(rows):
        scale = scale.repeat_interleave(BLOCK, 0)[: x.data.shape[0]]
    if tuple(scale.shape) != (*rows, _blocks(k)):
        raise ValueError(f"scales {tuple(x.scale.shape)} do not belong to values {tuple(x.data.shape)}")
    return (x.data.float() * scale.repeat_interleave(BLOCK, -1)[..., :k]).to(dtype)


def fp8_matmul(a: BlockFp8, b: BlockFp8, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a b^T`` ``[..., N]`` of ``a`` ``[..., K]`` (:func:`quantize_rows`) and ``b`` ``[N, K]``
    (:func:`quantize_weight`), fp32 sums, rounded once to ``out_dtype`` (bf16, fp16 or fp32).

    K is a multiple of 16; a single row of ``a`` is the form for one token.  Not differentiable."""
    if _lib.eager(*a, *b) and (out := _lib.native().fp8_matmul(*a, *b, out_dtype)) is not None:
        return out
    a, b = BlockFp8(*a), BlockFp8(*b)
    _check_blocks("a", a)
    _check_blocks("b", b, two_dim=True)
    if out_dtype not in (*_HALF, torch.float32):
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    k, rows = a.data.shape[-1], a.data.shape[:-1]
    if b.data.shape[1] != k:
        raise ValueError(f"a [..., K] and b [N, K] expected, got {tuple(a.data.shape)} and {tuple(b.data.shape)}")
    if tuple(a.scale.shape) != (*rows, _blocks(k)) or tuple(b.scale.shape) != (_blocks(b.data.shape[0]), _blocks(k)):
        raise ValueError(f"scales {tuple(a.scale.shape)} and {tuple(b.scale.shape)} do not belong to values "
                         f"{tuple(a.data.shape)} and {tuple(b.data.shape)}")
    _check_gpu("a and b", *a, *b)
    out = _ops().matmul8(a.data.reshape(-1, k), a.scale.reshape(-1, _blocks(k)), b.data, b.scale, out_dtype)
    return out.view(*rows, b.data.shape[0])


# ------------------------------------------------------------------- norm
def _check_norm(x, delta, of):
    _check_operand("x", x, of=of)
    if x.shape[-1] > 8192:
        raise ValueError(f"x's last dimension must be at most 8192, got {x.shape[-1]}")
    if delta is not None and (delta.shape != x.shape or delta.dtype != x.dtype or delta.device != x.device):
        raise ValueError("x and delta must have one shape, type and device")


def add_rms_norm_fp8(x: torch.Tensor, delta: torch.Tensor | None = None, eps: float = 1e-6):
    """``(s, y)``: ``s = x + delta`` rounded to its type (``x`` itself without ``delta``) and
    ``y = s / rms(s)`` (no weight) as :class:`BlockFp8` rows, in one pass; the row's sum of squares, its root and
    ``y`` before the rounding are fp32.

    ``x`` ``[..., D]`` bf16 or fp16, D a multiple of 16 up to 8192.  Not differentiable: training goes through
    :func:`norm_projection`."""
    if _lib.eager(x, delta) and (got := _lib.native().add_rms_norm_fp8(x, delta, eps)) is not None:
        return got[0], BlockFp8(*got[1:])
    _check_norm(x, delta, 16)
    _check_gpu("x", x)
    d = x.shape[-1]
    s, y, scale, _ = _ops().norm8(x.detach().reshape(-1, d), None if delta is None else delta.detach().reshape(-1, d),
                                  float(eps))
    return (x if delta is None else s.view(x.shape)), BlockFp8(y.view(x.shape), scale.view(*x.shape[:-1], _blocks(x.shape[-1])))


# ------------------------------------------------------- differentiable forms
def _check_weights(x, weights, k):
    if not 1 <= len(weights) <= 4:
        raise ValueError(f"1 to 4 weights are expected, got {len(weights)}")
    for w in weights:
        if w.dim() != 2 or w.shape[1] != k or w.shape[0] < 8 or w.shape[0] % 8:
            raise ValueError(f"a weight must be [N, {k}], N a multiple of 8, got {tuple(w.shape)}")
        if w.dtype != x.dtype or w.device != x.device:
            raise ValueError(f"a weight must have the operand's type and device ({x.dtype}, {x.device}), got {w.dtype}, "
                             f"{w.device}")


def _stacked(parts, dim):
    """Parts that the kernels can take side by side: whole blocks, or one part."""
    if len(parts) > 1 and any(p.shape[dim] % BLOCK for p in parts[:-1]):
        return [torch.cat(parts, dim)]
    return list(parts)


def _product(ops, x8, xs, weights, transpose, dtype):
    """x W^T for the stacked weights, and the weights' transposed blocks."""
    w8, ws, wt, wts = ops.quant_weight8(_stacked(weights, 0), transpose)
    return ops.matmul8(x8, xs, w8, ws, dtype), wt, wts


def _split(y, shape, weights):
    """y's columns by weight, in the operand's leading shape."""
    out, at = [], 0
    for w in weights:
        out.append(y[:, at:at + w.shape[0]].view(*shape, w.shape[0]))
        at += w.shape[0]
    return out


def _cotangents(dys, sizes, like):
    """The outputs' gradients as matrices of one type; zeros for an output that did not reach the loss."""
    return [like.new_zeros((like.shape[0], n)) if d is None else d.reshape(-1, n) for d, n in zip(dys, sizes)]


def _between(dtype):
    """The type of a gradient between two kernels: fp16, whose own rounding (2^-11) a second one would be felt beside, goes
    through fp32; bf16 stays (half the bytes, an error of 1.4 times one rounding's)."""
    return torch.float32 if dtype == torch.float16 else dtype


def _backward_products(ctx, dys, x8, xs, wt, wts, want_x, want_w, dtype):
    """(gradient of the 8-bit operand in ``dtype``, gradients of the weights)."""
    ops = torch.ops.kdattn
    dx, dws, at = None, [], 0
    parts = _stacked(dys, 1)
    if want_x:
        d8, ds = ops.quant_rows8(parts)
        dx = ops.matmul8(d8, ds, wt, wts, dtype, True)
    dw = ops.weight_grad8(parts, x8, xs, ctx.k) if any(want_w) else None
    for d, want in zip(dys, want_w):
        dws.append(dw[at:at + d.shape[1]] if want else None)
        at += d.shape[1]
    return dx, dws


class _NormProjection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, eps, *weights):
        ops, k, shape = torch.ops.kdattn, x.shape[-1], x.shape[:-1]
        s, y8, ys, rstd = ops.norm8(x.reshape(-1, k), None if delta is None else delta.reshape(-1, k), eps)
        want_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        y, wt, wts = _product(ops, y8, ys, weights, want_x, x.dtype)
        ctx.save_for_backward(y8, ys, rstd, wt, wts)
        ctx.k, ctx.dtype, ctx.sizes, ctx.shape = k, x.dtype, [w.shape[0] for w in weights], x.shape
        ctx.set_materialize_grads(False)
        return (None if delta is None else s.view(x.shape), *_split(y, shape, weights))

    @staticmethod
    @once_differentiable
    def backward(ctx, dsum, *dys):
        y8, ys, rstd, wt, wts = ctx.saved_tensors
        want_x, want_d = ctx.needs_input_grad[:2]
        none = [None] * len(dys)
        if all(d is None for d in dys):  # the products did not reach the loss
            return (dsum if want_x else None, dsum if want_d else None, None, *none)
        given = next(d for d in dys if d is not None)
        dys = _cotangents(dys, ctx.sizes, given.new_empty((y8.shape[0], 0)))
        g, dws = _backward_products(ctx, dys, y8, ys, wt, wts, want_x or want_d, ctx.needs_input_grad[3:],
                                    _between(ctx.dtype))
        dx = None
        if g is not None:
            dx = torch.ops.kdattn.norm8_bwd(g, None if dsum is None else dsum.reshape(-1, ctx.k), y8, ys, rstd,
                                               ctx.dtype).view(ctx.shape)
        return (dx if want_x else None, dx if want_d else None, None, *dws)


def norm_projection(x: torch.Tensor, delta: torch.Tensor | None, *weights: torch.Tensor, eps: float = 1e-6):
    """``(s, y_1, ...)``: ``s = x + delta`` (``x`` itself where ``delta`` is None) and ``y_i = rms_norm(s) W_i^T``, the
    normalised rows and the weights in 8-bit blocks.

    ``x``, ``delta`` ``[..., K]`` and 1 to 4 ``weights`` ``[N_i, K]``, bf16 or fp16 of one type; K (up to 8192) and N_i
    multiples of 8.  The weights' blocks are those of all weights stacked.  Differentiable once; the backward
    keeps the normalised rows in 8 bits and one float a row.  The y_i are columns of one product, strided."""
    if _lib.eager(x, delta, *weights) and (got := _lib.native().norm_projection(x, delta, weights, eps)) is not None:
        return tuple(got)
    _check_norm(x, delta, 8)
    _check_weights(x, weights, x.shape[-1])
    _check_gpu("x", x)
    _ops()
    s, *y = _NormProjection.apply(x, delta, float(eps), *weights)
    return (x if delta is None else s, *y)


class _Projection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        ops, k = torch.ops.kdattn, x.shape[-1]
        x8, xs = ops.quant_rows8([x.reshape(-1, k)])
        y, wt, wts = _product(ops, x8, xs, [weight], ctx.needs_input_grad[0], x.dtype)
        ctx.save_for_backward(x8, xs, wt, wts)
        ctx.k, ctx.dtype, ctx.shape = k, x.dtype, x.shape
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x8, xs, wt, wts = ctx.saved_tensors
        dx, (dw,) = _backward_products(ctx, [dy.reshape(-1, dy.shape[-1])], x8, xs, wt, wts, *ctx.needs_input_grad[:1],
                                       ctx.needs_input_grad[1:], ctx.dtype)
        return None if dx is None else dx.view(ctx.shape), dw


def fp8_projection(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``x W^T`` of ``x`` ``[..., K]`` and ``weight`` ``[N, K]`` (bf16 or fp16; K, N multiples of 8) with both in
    8-bit blocks.  Differentiable once; the backward keeps ``x`` in 8 bits."""
    if _lib.eager(x, weight) and (y := _lib.native().fp8_projection(x, weight)) is not None:
        return y
    _check_operand("x", x)
    _check_weights(x, [weight], x.shape[-1])
    _check_gpu("x", x)
    _ops()
    return _Projection.apply(x, weight)


class _SwigluProjection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, weight):
        ops, h = torch.ops.kdattn, a.shape[-1]
        want = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        y8, ys, a8, a_s, b8, b_s = ops.gate8(a.reshape(-1, h), b.reshape(-1, h), want)
        y, wt, wts = _product(ops, y8, ys, [weight], want, a.dtype)
        ctx.save_for_backward(y8, ys, a8, a_s, b8, b_s, wt, wts)
        ctx.k, ctx.dtype, ctx.shape = h, a.dtype, a.shape
        return y.view(*a.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        y8, ys, a8, a_s, b8, b_s, wt, wts = ctx.saved_tensors
        want_a, want_b, want_w = ctx.needs_input_grad
        g, (dw,) = _backward_products(ctx, [dy.reshape(-1, dy.shape[-1])], y8, ys, wt, wts, want_a or want_b, [want_w],
                                     _between(ctx.dtype))
        da = db = None
        if g is not None:
            da, db = (t.view(ctx.shape) for t in torch.ops.kdattn.gate8_bwd(g, a8, a_s, b8, b_s, ctx.dtype))
        return da if want_a else None, db if want_b else None, dw


def swiglu_projection(a: torch.Tensor, b: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``(silu(a) b) W^T`` of ``a``, ``b`` ``[..., H]`` and ``weight`` ``[N, H]`` (bf16 or fp16; H, N multiples of 8),
    the gated rows and the weight in 8-bit blocks.  Differentiable once; the backward keeps ``a``, ``b`` and the
    gated rows in 8 bits each."""
    if _lib.eager(a, b, weight) and (y := _lib.native().swiglu_projection(a, b, weight)) is not None:
        return y
    _check_operand("a", a)
    if b.shape != a.shape or b.dtype != a.dtype or b.device != a.device:
        raise ValueError("a and b must have one shape, type and device")
    _check_weights(a, [weight], a.shape[-1])
    _check_gpu("a", a)
    _ops()
    return _SwigluProjection.apply(a, b, weight)


__all__ = ["BLOCK", "BlockFp8", "quantize_rows", "quantize_weight", "dequantize", "fp8_matmul", "add_rms_norm_fp8",
           "norm_projection", "fp8_projection", "swiglu_projection"]
