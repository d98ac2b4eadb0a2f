"""A linear layer in 8 bits, y = x W^T, for training and serving: block quantisation (:func:`qgemm_b200.quantize_block`) and
the product whose power-of-two scales the tensor cores apply (:func:`qgemm_b200.fp8_block_mm_e8m0`), run together.

With Q the quantisation to FP8 e4m3 over blocks of 128 along the axis a product sums over (squares of 128 x 128 for W):

    forward   y  = Q(x) Q(W)^T                    sums over the input features
    backward  dx = Q(dy) Q(W)                     sums over the output features; the squares' codes are the same transposed
              dW = Q(dy^T) Q(Q(x)^T)^T            sums over the tokens

What the forward pass saves of x is Q(x), one byte an element plus 1/128: the codes its own product read. The backward pass
makes the operand of dW from them, quantised anew along the tokens (:func:`qgemm_b200.requantize_block`), so training keeps
no 16- or 32-bit copy of the activation. All sums are fp32, made as :func:`qgemm_b200.fp8_block_mm_e8m0` says; y, dx have
x's type and dW has W's, each rounded once.

Gradients pass through Q as through the identity. The reference has no layer and no backward pass; its ``fp8_mm(a, b, as, bs,
c)`` (src/mix_gemm/hip_mix_gemm_kernel.cpp:508-516) is the forward product alone.
"""
from __future__ import annotations

from contextlib import nullcontext
from dataclasses import dataclass, field

import torch
from torch.autograd import forward_ad

from . import (BLOCK, ERR_INVALID_ARG, ERR_UNSUPPORTED, QgemmError, _dtype_code, _launch, _matrix, _quantize_block,
               _scale_block_rows, _written)

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class _Form:
    """Where a row-form [rows, cols] matrix lies in a buffer of bytes: codes at ``codes`` with leading dimension ``ld``, scales
    at ``scale``; ``end`` is where the next may start. A layer call keeps all its quantised matrices in one or two buffers:
    for short calls making the tensors costs more than the GPU takes for them."""
    __slots__ = ("rows", "cols", "block_rows", "codes", "ld", "scale", "end")

    def __init__(self, start: int, rows: int, cols: int, square: bool = False):
        self.rows, self.cols, self.block_rows = rows, cols, BLOCK if square else 1
        self.codes, self.ld = start, (cols + 15) & -16
        self.scale = (start + rows * self.ld + 127) & -128
        self.end = (self.scale + self._scales() + 127) & -128

    def _scales(self) -> int:
        return -(-self.cols // BLOCK) * -(-self.rows // self.block_rows)

    def tensors(self, buffer):
        """(codes, scales) as tensors that share the buffer's memory."""
        q = buffer[self.codes:self.codes + self.rows * self.ld].view(_E4M3).view(self.rows, self.ld)[:, :self.cols]
        s = buffer[self.scale:self.scale + self._scales()].view(_E8M0)
        return q, s.view(-(-self.cols // BLOCK), -(-self.rows // self.block_rows))


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
    """What :func:`fp8_linear_forward` keeps for :func:`fp8_linear_backward`. :attr:`x` is the 8-bit checkpoint of the layer's
    input, ``(codes, scales)`` of [tokens, in] (:func:`qgemm_b200.dequantize_block` restores it); None if no gradient of the
    weight was asked for."""
    buffer: torch.Tensor | None  # x's codes, and the transposed weight's unless that is a packed one's
    x_form: _Form | None
    weight_form: _Form | None
    weight_t: tuple | None  # (codes, scales) of a packed weight's transpose
    x_shape: tuple
    x_dtype: torch.dtype
    weight_dtype: torch.dtype | None
    out_features: int
    device: torch.device = field(default=None)
    stream: int = 0  # the forward call's, to which the buffer's memory belongs

    @property
    def x(self):
        return None if self.x_form is None else self.x_form.tensors(self.buffer)


def pack_weight(weight, backward: bool = False) -> PackedWeight:
    """Quantises a weight [out, in] for :func:`fp8_linear` once; ``backward`` keeps its transpose too, so that gradients
    with respect to x can be taken (the weight itself gets none)."""
    if weight.dim() != 2:
        raise QgemmError(ERR_INVALID_ARG, "a weight is [out, in]")
    if weight.dtype not in _TYPES:
        raise QgemmError(ERR_UNSUPPORTED, f"a weight of dtype {weight.dtype}")
    w = _rows(weight.detach())
    return PackedWeight(*_quantize_block(w, *_matrix("weight", w), True, True, backward))


def _rows(t):
    """The same matrix with unit inner stride and rows that do not overlap (broadcast gradients are made whole)."""
    if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]):
        return t
    # an empty matrix counts as contiguous whatever its strides
    return t.contiguous() if t.numel() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _tokens(shape) -> int:
    tokens = 1
    for d in shape[:-1]:
        tokens *= d
    return tokens


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


def _quantize(device, t, base: int, row: _Form | None, column: _Form | None, square: bool = False) -> None:
    """Quantises the matrix t into the forms of the buffer at address ``base``."""
    rows, cols, ld = _matrix("matrix", t)
    r = (base + row.codes, row.ld, base + row.scale) if row is not None else (None, 0, None)
    c = (base + column.codes, column.ld, base + column.scale) if column is not None else (None, 0, None)
    _launch("qgemm_quantize_block", device, _dtype_code(t), t.data_ptr(), ld, rows, cols, BLOCK if square else 1, *r, *c)


def _product(device, a, b, c, m: int, n: int, k: int, accumulate: bool = False) -> None:
    """c = a b^T; a and b: (address of codes, leading dimension, address of scales, rows a scale covers)."""
    _, _, ldc = _matrix("c", c)
    _launch("qgemm_fp8_block_e8m0_gemm", device, _dtype_code(c), a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3],
            1 if accumulate else 0, c.data_ptr(), ldc, m, n, k)


def _at(form: _Form, base: int):
    return base + form.codes, form.ld, base + form.scale, form.block_rows


def _of(codes, scale):
    rows, cols, ld = _matrix("codes", codes)
    return codes.data_ptr(), ld, scale.data_ptr(), _scale_block_rows("scale", scale, rows, cols, codes.device)


def fp8_linear_forward(x, weight, need_dx: bool = True, need_dw: bool = True, out_dtype=None):
    """``(y, saved)``: y = x W^T of x [..., in] and ``weight`` [out, in] (a bf16 / fp16 / fp32 matrix, quantised in this
    call, or a :class:`PackedWeight`), without autograd. ``saved`` holds what the gradients that are needed take."""
    packed = isinstance(weight, PackedWeight)
    if not packed and (weight.dim() != 2 or weight.dtype not in _TYPES):
        raise QgemmError(ERR_INVALID_ARG, "a weight is a bf16, fp16 or fp32 matrix [out, in], or a PackedWeight")
    device = x.device
    if weight.device != device:
        raise QgemmError(ERR_INVALID_ARG, "x and the weight are on different devices")
    out_features, in_features = weight.shape
    x2 = _flat(x, in_features, "x")
    tokens = x2.shape[0]
    if packed:
        if need_dw:
            raise QgemmError(ERR_INVALID_ARG, "a PackedWeight has no gradient: need_dw=False")
        if need_dx and weight.codes_t is None:
            raise QgemmError(ERR_INVALID_ARG, "gradients with respect to x need pack_weight(..., backward=True)")
    # kept for the backward pass: x's codes, the weight's transpose; behind them what only this call needs
    at = 0
    x_form = w_form = wt_form = None
    if need_dw:
        x_form = _Form(0, tokens, in_features)
        at = x_form.end
    if need_dx and not packed:
        wt_form = _Form(at, in_features, out_features, True)
        at = wt_form.end
    kept = at
    if x_form is None:
        x_form = _Form(at, tokens, in_features)
        at = x_form.end
    if not packed:
        w_form = _Form(at, out_features, in_features, True)
        at = w_form.end
    buffer = torch.empty(kept, dtype=torch.uint8, device=device) if need_dw or wt_form is not None else None
    scratch = torch.empty(at - kept, dtype=torch.uint8, device=device) if at > kept else None
    base = buffer.data_ptr() if buffer is not None else 0
    scratch_base = scratch.data_ptr() - kept if at > kept else 0
    x_base = base if need_dw else scratch_base
    if packed:
        w_at = _of(weight.codes, weight.scale)
    else:
        w = _rows(weight.detach() if weight.requires_grad else weight)
        rows, cols, ld = _matrix("weight", w)
        turned = (base + wt_form.codes, wt_form.ld, base + wt_form.scale) if wt_form is not None else (None, 0, None)
        _launch("qgemm_quantize_block", device, _dtype_code(w), w.data_ptr(), ld, rows, cols, BLOCK,
                scratch_base + w_form.codes, w_form.ld, scratch_base + w_form.scale, *turned)
        w_at = _at(w_form, scratch_base)
    _quantize(device, x2, x_base, x_form, None)
    y = torch.empty((tokens, out_features), dtype=out_dtype or x.dtype, device=device)
    _product(device, _at(x_form, x_base), w_at, y, tokens, out_features, in_features)
    saved = LinearSaved(buffer, x_form if need_dw else None, wt_form,
                        (weight.codes_t, weight.scale_t) if packed and need_dx else None, tuple(x.shape), x.dtype,
                        None if packed else weight.dtype, out_features, device,
                        torch._C._cuda_getCurrentRawStream(device.index))
    return (y if x.dim() == 2 else y.view(*x.shape[:-1], out_features)), saved


def fp8_linear_backward(dy, saved: LinearSaved, dw=None, accumulate: bool = False):
    """``(dx, dw)`` from dy [..., out] and what the forward call saved; None for a gradient it saved nothing for. ``dw``: a
    matrix [out, in] to write into instead of a new one, or with ``accumulate`` (fp32) to add to, as over the micro-batches
    of one step. It may run on another stream than the forward call, once that stream waits for it; ``saved`` may then be
    dropped at once."""
    out_features, in_features = saved.out_features, saved.x_shape[-1]
    dy2 = _flat(dy, out_features, "dy")
    device = saved.device
    need_dx, need_dw = saved.weight_form is not None or saved.weight_t is not None, saved.x_form is not None
    tokens = _tokens(saved.x_shape)
    if dy2.shape[0] != tokens:
        raise QgemmError(ERR_INVALID_ARG, f"dy has {dy2.shape[0]} rows, x had {tokens}")
    if dy.device != device:
        raise QgemmError(ERR_INVALID_ARG, "dy is on another device than the layer")
    if accumulate and dw is None:
        raise QgemmError(ERR_INVALID_ARG, "accumulate adds to a given dw")
    if dw is not None:
        if not need_dw:
            raise QgemmError(ERR_INVALID_ARG, "the forward call saved nothing for dw")
        if dw.dim() != 2 or tuple(dw.shape) != (out_features, in_features) or dw.device != device:
            raise QgemmError(ERR_INVALID_ARG, f"dw is [{out_features}, {in_features}] on the layer's device")
        _matrix("dw", dw)
        if accumulate and dw.dtype != torch.float32:
            raise QgemmError(ERR_UNSUPPORTED, "accumulate needs a fp32 dw")
    if not need_dx and not need_dw:
        return None, None
    at = 0
    along = across = x_across = None
    if need_dx:
        along = _Form(at, tokens, out_features)
        at = along.end
    if need_dw:
        across = _Form(at, out_features, tokens)
        x_across = _Form(across.end, in_features, tokens)
        at = x_across.end
    scratch = torch.empty(at, dtype=torch.uint8, device=device)
    base = scratch.data_ptr()
    kept = 0
    if saved.buffer is not None:
        kept = saved.buffer.data_ptr()
        if torch._C._cuda_getCurrentRawStream(device.index) != saved.stream:
            # nobody else knows of this use: without it the memory could be given out again before these kernels are done
            saved.buffer.record_stream(torch.cuda.current_stream(device))
    _quantize(device, dy2, base, along, across)
    dx = None
    if need_dx:
        dx = torch.empty((tokens, in_features), dtype=saved.x_dtype, device=device)
        w_at = _at(saved.weight_form, kept) if saved.weight_form is not None else _of(*saved.weight_t)
        _product(device, _at(along, base), w_at, dx, tokens, in_features, out_features)
        if len(saved.x_shape) != 2:
            dx = dx.view(saved.x_shape)
    if need_dw:
        f = saved.x_form
        _launch("qgemm_requantize_block", device, kept + f.codes, f.ld, kept + f.scale, tokens, in_features,
                base + x_across.codes, x_across.ld, base + x_across.scale)
        given = dw is not None
        if not given:
            dw = torch.empty((out_features, in_features), dtype=saved.weight_dtype, device=device)
        _product(device, _at(across, base), _at(x_across, base), dw, out_features, in_features, tokens, accumulate)
        if given:
            _written(dw)
    return dx, dw


# Where the gradient of a leaf is gathered: its node belongs to the stream that was current when the node was made, and lives
# as long as any graph refers to the leaf. torch does not tell the stream, so the layer's calls write it into the node.
_STREAM = "qgemm_b200.linear: stream"
_PROBE = "qgemm_b200.linear: probe"


def _leaf_node(node):
    """The leaf's node that ``node`` leads to by way of at most four operations of one input each (casts, transposes), or
    None. A leaf's node is its own."""
    for _ in range(5):
        following = node.next_functions
        if not following and hasattr(node, "variable"):
            return node
        if len(following) != 1 or following[0][0] is None:
            return None
        node = following[0][0]
    return None


def _node(t):
    """The node that gathers or passes on t's gradient."""
    return t.view_as(t).grad_fn.next_functions[0][0] if t.is_leaf else t.grad_fn


def _probe_nodes(capturing: bool, *tensors) -> None:
    """Before a call on a stream other than the default one: refuses a capture whose backward pass would come to a node of
    the default stream, and writes into the nodes that live already that they do."""
    for t in tensors:
        if t is None or not t.requires_grad:
            continue
        # through a derived tensor's graph a node lives in any case: only a refusal looks there
        node = _node(t) if t.is_leaf else (_leaf_node(t.grad_fn) if capturing else None)
        if node is None:
            continue
        if capturing and node.metadata.get(_STREAM) == 0:
            del node  # the error's traceback must not keep it alive
            raise QgemmError(ERR_UNSUPPORTED, "capturing a graph while an earlier graph of the same leaves is alive")
        node.metadata[_PROBE] = True  # gone with the last reference to the node, here if no graph holds one


def _note_nodes(y, stream: int) -> None:
    """After a call: the nodes it made are its stream's. One that lived before and has no mark counts as the default stream's
    once a call there has met it."""
    for node, _ in y.grad_fn.next_functions:
        if node is not None and node.next_functions:
            node = _leaf_node(node) if stream == 0 else None
        if node is None:
            continue
        if stream == 0 or _PROBE not in node.metadata:
            node.metadata.setdefault(_STREAM, stream)


def _as_saved(buffer, weight_t):
    """A saved buffer and transposed weight as the kernels take them. Saved-tensor hooks (offloading to the host) give back
    equal tensors, but at any address and without the padding that starts a weight's rows on 16-byte boundaries."""
    if buffer is not None and (buffer.data_ptr() % 16 or not buffer.is_contiguous()):
        buffer = buffer.clone(memory_format=torch.contiguous_format)
    if not weight_t:
        return buffer, None
    codes, scale = weight_t
    rows, cols = codes.shape
    if codes.data_ptr() % 16 or codes.stride(0) % 16 or codes.stride(1) != 1:
        codes = torch.empty_strided((rows, cols), ((cols + 15) & -16, 1), dtype=codes.dtype, device=codes.device).copy_(codes)
    return buffer, (codes, scale.contiguous())


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, packed, out_dtype):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        y, saved = fp8_linear_forward(x, weight if packed is None else packed, need_dx, need_dw, out_dtype)
        ctx.save_for_backward(saved.buffer, *(saved.weight_t or ()))
        saved.buffer = saved.weight_t = None
        ctx.rest = saved
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        r = ctx.rest
        buffer, *weight_t = ctx.saved_tensors
        buffer, weight_t = _as_saved(buffer, weight_t)
        saved = LinearSaved(buffer, r.x_form, r.weight_form, weight_t, r.x_shape, r.x_dtype, r.weight_dtype, r.out_features,
                            r.device, r.stream)
        dx, dw = fp8_linear_backward(dy, saved)
        return dx, dw, None, None


def _refuse_tangents(*tensors) -> None:
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise QgemmError(ERR_UNSUPPORTED, "fp8_linear has no forward-mode derivative: its input carries a tangent")


def fp8_linear(x, weight, out_dtype=None):
    """y = x W^T in 8 bits with autograd: x [..., in] bf16 / fp16 / fp32, ``weight`` [out, in] a matrix that may require a
    gradient, or a :class:`PackedWeight` (serving; frozen layers). y has x's type unless ``out_dtype`` says otherwise.
    Gradients are reverse-mode only: a tensor that carries a forward-mode tangent is refused, with gradients enabled or not.
    Runs on the current stream of x's device. A CUDA graph is captured after one ordinary call on the device.

    A capture is refused while an earlier graph of the same leaves, made on the default stream, is alive: the leaves' gradient
    nodes then belong to that stream, and torch would leave the capture in the backward pass. The refusal sees x and the
    weight themselves, or their leaves through up to four one-input operations (casts, transposes), where an earlier call of
    this function on the default stream met them; a leaf that only other operations used there is not seen. (A node that
    other operations made on some other stream and a default-stream call of this function met counts as the default
    stream's.) Delete what keeps that graph alive, or capture :func:`fp8_linear_forward` and :func:`fp8_linear_backward`,
    which use no autograd."""
    packed = weight if isinstance(weight, PackedWeight) else None
    w = None if packed is not None else weight
    _refuse_tangents(x, w)
    if not torch.is_grad_enabled() or not (x.requires_grad or (w is not None and w.requires_grad)):
        return fp8_linear_forward(x, weight, False, False, out_dtype)[0]
    if not x.is_cuda:
        raise QgemmError(ERR_INVALID_ARG, "x must be a CUDA tensor (there is no CPU path)")
    stream = torch.cuda.current_stream(x.device).cuda_stream
    if stream != 0:  # the default stream is never captured
        with nullcontext() if torch.cuda.current_device() == x.device.index else torch.cuda.device(x.device):
            capturing = torch.cuda.is_current_stream_capturing()
        _probe_nodes(capturing, x, w)
    y = _Fp8Linear.apply(x, w, packed, out_dtype)
    _note_nodes(y, stream)
    return y
