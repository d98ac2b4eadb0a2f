"""A linear layer in 8 bits, y = x W^T, for training and serving: block quantisation (:func:`qgemm_b200.quantize_block`) and
the product whose power-of-two scales the tensor cores apply (:func:`qgemm_b200.fp8_block_mm_e8m0`), run together.

With Q the quantisation to FP8 e4m3 over blocks of 128 along the axis a product sums over (squares of 128 x 128 for W):

    forward   y  = Q(x) Q(W)^T                    sums over the input features
    backward  dx = Q(dy) Q(W)                     sums over the output features; the squares' codes are the same transposed
              dW = Q(dy^T) Q(Q(x)^T)^T            sums over the tokens

What the forward pass saves of x is Q(x), one byte an element plus 1/128: the codes its own product read. The backward pass
makes the operand of dW from them, quantised anew along the tokens (:func:`qgemm_b200.requantize_block`), so training keeps
no 16- or 32-bit copy of the activation. All sums are fp32; y, dx have x's type and dW has W's, each rounded once.

Gradients pass through Q as through the identity. The reference has no layer and no backward pass; its ``fp8_mm(a, b, as, bs,
c)`` (src/mix_gemm/hip_mix_gemm_kernel.cpp:508-516) is the forward product alone.
"""
from __future__ import annotations

from contextlib import nullcontext
from dataclasses import dataclass

import torch

from . import ERR_INVALID_ARG, ERR_UNSUPPORTED, QgemmError, _matrix, _quantize_block, fp8_block_mm_e8m0, requantize_block

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


@dataclass
class PackedWeight:
    """A weight [out, in] quantised once. ``codes_t`` / ``scale_t`` (its transpose, for dx) are None unless asked for."""
    codes: torch.Tensor
    scale: torch.Tensor
    codes_t: torch.Tensor | None = None
    scale_t: torch.Tensor | None = None

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device


@dataclass
class LinearSaved:
    """What :func:`fp8_linear_forward` keeps for :func:`fp8_linear_backward`. ``x_codes`` / ``x_scale`` are the 8-bit
    checkpoint of the layer's input, [tokens, in] (:func:`qgemm_b200.dequantize_block` restores it)."""
    x_codes: torch.Tensor | None
    x_scale: torch.Tensor | None
    weight_codes_t: torch.Tensor | None
    weight_scale_t: torch.Tensor | None
    x_shape: tuple
    x_dtype: torch.dtype
    weight_dtype: torch.dtype | None
    out_features: int


def pack_weight(weight, backward: bool = False) -> PackedWeight:
    """Quantises a weight [out, in] for :func:`fp8_linear` once; ``backward`` keeps its transpose too, so that gradients
    with respect to x can be taken (the weight itself gets none)."""
    if weight.dim() != 2:
        raise QgemmError(ERR_INVALID_ARG, "a weight is [out, in]")
    if weight.dtype not in _TYPES:
        raise QgemmError(ERR_UNSUPPORTED, f"a weight of dtype {weight.dtype}")
    return PackedWeight(*_quantized(_rows(weight.detach()), True, True, backward))


def _quantized(t, square: bool, row: bool, column: bool):
    return _quantize_block(t, *_matrix("matrix", t), square, row, column)


def _rows(t):
    """The same matrix with unit inner stride and rows that do not overlap (broadcast gradients are made whole)."""
    if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]):
        return t
    # an empty matrix counts as contiguous whatever its strides
    return t.contiguous() if t.numel() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _flat(x, features: int, what: str):
    if x.dim() < 1 or x.shape[-1] != features:
        raise QgemmError(ERR_INVALID_ARG, f"{what} is [..., {features}], got {list(x.shape)}")
    if not x.is_cuda:
        raise QgemmError(ERR_INVALID_ARG, f"{what} must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in _TYPES:
        raise QgemmError(ERR_UNSUPPORTED, f"{what} of dtype {x.dtype}")
    if x.requires_grad:
        x = x.detach()
    if x.dim() != 2:
        x = x.reshape(_tokens(x.shape), features)
    return _rows(x)


def _tokens(shape) -> int:
    tokens = 1
    for d in shape[:-1]:
        tokens *= d
    return tokens


def fp8_linear_forward(x, weight, need_dx: bool = True, need_dw: bool = True, out_dtype=None):
    """``(y, saved)``: y = x W^T of x [..., in] and ``weight`` [out, in] (a bf16 / fp16 / fp32 matrix, quantised in this
    call, or a :class:`PackedWeight`), without autograd. ``saved`` holds what the gradients that are needed take."""
    packed = isinstance(weight, PackedWeight)
    if not packed and (weight.dim() != 2 or weight.dtype not in _TYPES):
        raise QgemmError(ERR_INVALID_ARG, "a weight is a bf16, fp16 or fp32 matrix [out, in], or a PackedWeight")
    if weight.device != x.device:
        raise QgemmError(ERR_INVALID_ARG, "x and the weight are on different devices")
    out_features, in_features = weight.shape
    x2 = _flat(x, in_features, "x")
    if packed:
        if need_dw:
            raise QgemmError(ERR_INVALID_ARG, "a PackedWeight has no gradient: need_dw=False")
        if need_dx and weight.codes_t is None:
            raise QgemmError(ERR_INVALID_ARG, "gradients with respect to x need pack_weight(..., backward=True)")
        w, ws, wt, wts = weight.codes, weight.scale, weight.codes_t, weight.scale_t
    else:
        w, ws, *turned = _quantized(_rows(weight.detach()), True, True, need_dx)
        wt, wts = turned if turned else (None, None)
    xq, xs = _quantized(x2, False, True, False)
    y = torch.empty((x2.shape[0], out_features), dtype=out_dtype or x.dtype, device=x.device)
    fp8_block_mm_e8m0(xq, w, xs, ws, y)
    saved = LinearSaved(xq if need_dw else None, xs if need_dw else None, wt if need_dx else None, wts if need_dx else None,
                        tuple(x.shape), x.dtype, None if packed else weight.dtype, out_features)
    return (y if x.dim() == 2 else y.view(*x.shape[:-1], out_features)), saved


def fp8_linear_backward(dy, saved: LinearSaved, dw=None, accumulate: bool = False):
    """``(dx, dw)`` from dy [..., out] and what the forward call saved; None for a gradient it saved nothing for. ``dw``: a
    matrix [out, in] to write into instead of a new one, or with ``accumulate`` (fp32) to add to, as over the micro-batches
    of one step."""
    dy2 = _flat(dy, saved.out_features, "dy")
    in_features = saved.x_shape[-1]
    need_dx, need_dw = saved.weight_codes_t is not None, saved.x_codes is not None
    tokens = _tokens(saved.x_shape)
    if dy2.shape[0] != tokens:
        raise QgemmError(ERR_INVALID_ARG, f"dy has {dy2.shape[0]} rows, x had {tokens}")
    kept = saved.x_codes if need_dw else saved.weight_codes_t
    if kept is not None and kept.device != dy.device:
        raise QgemmError(ERR_INVALID_ARG, "dy is on another device than the layer")
    if accumulate and dw is None:
        raise QgemmError(ERR_INVALID_ARG, "accumulate adds to a given dw")
    if dw is not None and not need_dw:
        raise QgemmError(ERR_INVALID_ARG, "the forward call saved nothing for dw")
    if not need_dx and not need_dw:
        return None, None
    forms = _quantized(dy2, False, need_dx, need_dw)
    dx = None
    if need_dx:
        dx = torch.empty((tokens, in_features), dtype=saved.x_dtype, device=dy.device)
        fp8_block_mm_e8m0(forms[0], saved.weight_codes_t, forms[1], saved.weight_scale_t, dx)
        dx = dx.view(saved.x_shape)
    if need_dw:
        xt, xts = requantize_block(saved.x_codes, saved.x_scale)
        if dw is None:
            dw = torch.empty((saved.out_features, in_features), dtype=saved.weight_dtype, device=dy.device)
        fp8_block_mm_e8m0(forms[-2], xt, forms[-1], xts, dw, accumulate=accumulate)
    return dx, dw


_STREAM = "qgemm_b200.linear stream"


def _accumulators(*leaves):
    """The nodes that end a graph at those of the tensors that are leaves with a gradient."""
    return [torch.autograd.graph.get_gradient_edge(t).node for t in leaves
            if t is not None and t.requires_grad and t.is_leaf]


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, packed, out_dtype):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        y, saved = fp8_linear_forward(x, weight if packed is None else packed, need_dx, need_dw, out_dtype)
        ctx.save_for_backward(saved.x_codes, saved.x_scale, saved.weight_codes_t, saved.weight_scale_t)
        saved.x_codes = saved.x_scale = saved.weight_codes_t = saved.weight_scale_t = None
        ctx.rest = saved
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        r = ctx.rest
        saved = LinearSaved(*ctx.saved_tensors, r.x_shape, r.x_dtype, r.weight_dtype, r.out_features)
        dx, dw = fp8_linear_backward(dy, saved)
        return dx, dw, None, None


def fp8_linear(x, weight, out_dtype=None):
    """y = x W^T in 8 bits with autograd: x [..., in] bf16 / fp16 / fp32, ``weight`` [out, in] a matrix that may require a
    gradient, or a :class:`PackedWeight` (serving; frozen layers). y has x's type unless ``out_dtype`` says otherwise.
    Runs on the current stream of x's device. A CUDA graph is captured after one ordinary call on the device. A leaf that an
    earlier layer call's graph, still alive, refers to is refused in a capture: its gradient node belongs to that call's
    stream, and torch would leave the capture in the backward pass. Delete what keeps that graph alive, or capture
    :func:`fp8_linear_forward` and :func:`fp8_linear_backward`, which use no autograd."""
    packed = weight if isinstance(weight, PackedWeight) else None
    w = None if packed is not None else weight
    if not torch.is_grad_enabled() or not (x.requires_grad or (w is not None and w.requires_grad)):
        return fp8_linear_forward(x, weight, False, False, out_dtype)[0]
    if not x.is_cuda:
        raise QgemmError(ERR_INVALID_ARG, "x must be a CUDA tensor (there is no CPU path)")
    stream = torch.cuda.current_stream(x.device).cuda_stream
    with nullcontext() if torch.cuda.current_device() == x.device.index else torch.cuda.device(x.device):
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing and any(n.metadata.get(_STREAM, stream) != stream for n in _accumulators(x, w)):
        raise QgemmError(ERR_UNSUPPORTED, "capturing a graph while an earlier graph of the same leaves is alive")
    y = _Fp8Linear.apply(x, w, packed, out_dtype)
    for node in _accumulators(x, w):  # alive as long as a graph refers to the leaf, and its marks with it
        node.metadata.setdefault(_STREAM, stream)
    return y
