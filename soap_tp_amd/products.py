"""Products of the layers whose weights SOAP trains: grouped by expert, from 8-bit activation
checkpoints, and in 8-bit integers.

The reference starts from a gradient matrix.  These are the products of a layer's forward and
backward pass up to that matrix, on the same library (``include/soap_mi355.h``) and in the same
manner as ``soap_tp_amd.ops``: device tensors only, work is enqueued on torch's current stream of the
tensors' device and never synchronised, bad arguments raise ``ValueError`` before anything is launched.

Tokens are rows.  With experts, the rows are sorted by expert and ``ends`` (int64, on the device) holds
for each expert the first row behind its own: expert ``e`` has the rows ``ends[e-1] .. ends[e]-1``.  An
expert may have no row, and the buffer may have rows behind the last expert's.  The sizes stay on the
device, so nothing here depends on their values on the host and calls can be captured into a graph.
Weights are (outputs, inputs) matrices, ``(experts, outputs, inputs)`` with experts; a dense layer
passes ``ends=None`` and two-dimensional weights.  Inputs are bfloat16, float16 or float32, rows may be
strided, sums are formed in float32 on the matrix cores.  An input whose rows are not contiguous (a transposed
matrix or stack of weights) is copied first, on every call.

    y  = expert_product(x, weights, ends)                   # y[t] = W_e x[t]
    dx = expert_input_gradient(dy, weights, ends)           # dx[t] = W_e^T dy[t]
    dw = expert_weight_gradient(dy, x, ends)                # dW_e = sum of dy[t] x[t]^T, float32
    update = soap_step(dw[e], state[e], ...)

``expert_linear`` is the first of them for autograd, with the other two as its backward pass.  No other call
here is recorded by autograd: its result requires no gradient, whatever its inputs do.  A tensor given as
``out`` counts as modified in place, and may require a gradient under ``torch.no_grad`` only.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from .ops._common import native_call, native_library, require_device_tensor, scratch

__all__ = [
    "ActivationCheckpoint",
    "checkpoint_activations",
    "expert_input_gradient",
    "expert_linear",
    "expert_product",
    "expert_weight_gradient",
    "int8_product",
    "quantize_tokens",
    "restore_activations",
]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
CHECKPOINT_BLOCK = 128  # columns that share an exponent
_INT8_MAX_INNER = 131071  # 16384 times more of them would leave 32-bit sums


class ActivationCheckpoint(NamedTuple):
    """A matrix kept in 8 bits: ``codes`` (int8, its shape) and ``exponents`` (uint8, one for each row
    and 128 columns); the values are ``codes * 2 ** (exponents - 127)``, NaN where the exponent is 255.
    ``dtype`` is the type of the matrix it was made from."""

    codes: Tensor
    exponents: Tensor
    dtype: torch.dtype


# ---- checks --------------------------------------------------------------------------------
#
# A small product takes the device less time than a line-by-line description of its arguments takes the
# host, so the checks that pass read each property once and messages are made only where one fails.

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _launch(index: int, name: str, *arguments) -> None:
    """Call an entry point on torch's current stream of device ``index``."""
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _launch(index, name, *arguments)
    native_call(name, *arguments, torch.cuda.current_stream(index).cuda_stream if _raw_stream is None else _raw_stream(index))


def _refuse_devices(device: torch.device, **tensors: Optional[Tensor]) -> None:
    for name, tensor in tensors.items():
        if tensor is not None:
            if tensor.device != device:
                raise ValueError(f"{name} is on {tensor.device}, expected {device}.")
            require_device_tensor(name, tensor)


def _check_matrix(name: str, tensor: Tensor, dimensions: int = 2) -> None:
    if not isinstance(tensor, Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(tensor).__name__}.")
    if tensor.ndim != dimensions:
        raise ValueError(f"{name} must be {dimensions}D, got {tensor.ndim}D.")


def _check_values(name: str, tensor: Tensor, dimensions: int = 2) -> int:
    """The code of the tensor's type."""
    _check_matrix(name, tensor, dimensions)
    code = _DTYPES.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{name} must use float32, bfloat16 or float16, got {tensor.dtype}.")
    return code


def _rows(tensor: Tensor) -> Tuple[Tensor, int]:
    """The tensor with its last dimension contiguous (copied if it is not) and its row stride."""
    rows, columns = tensor.shape[-2:]
    strides = tensor.stride()
    if rows <= 1:
        if columns <= 1 or strides[-1] == 1:
            return tensor, max(1, columns)
    elif strides[-2] >= max(1, columns) and (columns <= 1 or strides[-1] == 1):
        return tensor, strides[-2]
    return tensor.contiguous(), max(1, columns)


def _experts(tensor: Tensor) -> Tuple[Tensor, int, int]:
    """Weights as (tensor, row stride, expert stride)."""
    tensor, row = _rows(tensor)
    return tensor, row, tensor.stride(0) if tensor.ndim == 3 and tensor.size(0) > 1 else 0


def _check_ends(ends: Optional[Tensor], experts: int) -> int:
    if ends is None:
        return 0
    _check_matrix("ends", ends, 1)
    if ends.dtype != torch.int64:
        raise ValueError(f"ends must use int64, got {ends.dtype}.")
    if ends.numel() != experts:
        raise ValueError(f"ends has {ends.numel()} entries, expected one for each of {experts} experts.")
    if experts > 1 and ends.stride(0) != 1:
        raise ValueError("ends must be contiguous.")
    return ends.data_ptr()


def _spans(tensor: Tensor) -> Tuple[int, int]:
    """First and last byte of memory that a tensor's elements use."""
    first = tensor.data_ptr()
    reach = sum((size - 1) * stride for size, stride in zip(tensor.shape, tensor.stride()))
    return first, first + (reach + 1) * tensor.element_size()


def _apart(a: Tensor, b: Tensor) -> bool:
    """Whether two tensors share no element: their memory does not meet, or they are different columns of
    rows with the same stride."""
    (first, last), (low, high) = _spans(a), _spans(b)
    if last <= low or high <= first:
        return True
    if a.ndim != 2 or b.ndim != 2 or a.stride(1) != 1 or b.stride(1) != 1:
        return False
    stride = a.stride(0) * a.element_size()
    if stride <= 0 or stride != b.stride(0) * b.element_size():
        return False
    shift = (low - first) % stride
    return shift >= a.size(1) * a.element_size() and stride - shift >= b.size(1) * b.element_size()


def _check_out(out: Tensor, shape: Tuple[int, ...], dtypes: Tuple[torch.dtype, ...], **inputs: Optional[Tensor]) -> int:
    """``out`` as a caller gave it: rows of contiguous values, written in place, apart from the inputs.
    The code of its type."""
    _check_matrix("out", out, len(shape))
    if tuple(out.shape) != shape:
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {shape}.")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out must not require a gradient: the call is not recorded by autograd.")
    if out.dtype not in dtypes:
        raise ValueError(f"out must use {' or '.join(str(d) for d in dtypes)}, got {out.dtype}.")
    if out.numel():
        strides = out.stride()
        if (shape[-1] > 1 and strides[-1] != 1) or (shape[-2] > 1 and strides[-2] < shape[-1]):
            raise ValueError("out must have contiguous rows that do not overlap.")
        if len(shape) == 3 and shape[0] > 1 and strides[0] < (shape[1] - 1) * _row_stride(out) + shape[2]:
            raise ValueError("out must have matrices that do not overlap.")
        for name, tensor in inputs.items():
            if tensor is not None and tensor.numel() and not _apart(out, tensor):
                raise ValueError(f"out must not overlap {name}.")
    return _DTYPES[out.dtype]


# The kernels write through addresses, which autograd does not see: a tensor that it saved for a backward pass
# has to be known as modified.
_modified = torch.autograd.graph.increment_version


def _row_stride(tensor: Tensor) -> int:
    return tensor.stride(-2) if tensor.size(-2) > 1 else max(1, tensor.size(-1))


def _out_types(dtype: torch.dtype) -> Tuple[torch.dtype, ...]:
    return (dtype,) if dtype == torch.float32 else (dtype, torch.float32)


# ---- grouped products ----------------------------------------------------------------------


def _grouped(x: Tensor, weights: Tensor, ends: Optional[Tensor], out: Optional[Tensor], transposed: int, name: str) -> Tensor:
    code = _check_values(name, x)
    if _check_values("weights", weights, 2 if ends is None else 3) != code:
        raise ValueError(f"weights must use {x.dtype} as {name} does, got {weights.dtype}.")
    tokens, width = x.shape
    outputs, inputs = weights.shape[-2:]
    inner, columns = (outputs, inputs) if transposed else (inputs, outputs)
    if width != inner:
        raise ValueError(f"{name} has {width} columns, expected {inner}.")
    experts = 1 if ends is None else weights.size(0)
    pointer = _check_ends(ends, experts)
    fresh = out is None
    out_code = code if fresh else _check_out(out, (tokens, columns), _out_types(x.dtype), **{name: x}, weights=weights, ends=ends)
    index = x.get_device()
    if (index < 0 or weights.get_device() != index or (pointer and ends.get_device() != index)
            or (not fresh and out.get_device() != index)):
        _refuse_devices(x.device, **{name: x}, weights=weights, ends=ends, out=out)
    if fresh:
        out = torch.empty((tokens, columns), dtype=x.dtype, device=x.device)
    if tokens and columns:
        rows, ldx = _rows(x)
        matrices, ldw, stride_w = _experts(weights)
        _launch(index, "soapmi_expert_product", code, rows.data_ptr(), ldx, matrices.data_ptr(), ldw, stride_w, transposed,
                pointer, experts, tokens, outputs, inputs, out_code, out.data_ptr(), columns if fresh else _row_stride(out),
                1 if fresh else 0)
        if not fresh:
            _modified(out)
    return out


def expert_product(x: Tensor, weights: Tensor, ends: Optional[Tensor], *, out: Optional[Tensor] = None) -> Tensor:
    """``y[t] = W_e x[t]`` for every row ``t`` of every expert ``e``.

    ``x`` is (tokens, inputs), ``weights`` (experts, outputs, inputs) of the same type; the result is
    (tokens, outputs) of that type.  ``out`` receives the result instead of a new tensor and may be
    float32.  Rows of no expert are zero in a new tensor and left as they were in ``out``.  Not recorded
    by autograd: see ``expert_linear``."""
    return _grouped(x, weights, ends, out, 0, "x")


def expert_input_gradient(gradient: Tensor, weights: Tensor, ends: Optional[Tensor], *, out: Optional[Tensor] = None) -> Tensor:
    """``dx[t] = W_e^T dy[t]``: the gradient of ``expert_product``'s ``x`` from that of its result,
    (tokens, inputs) from (tokens, outputs); otherwise as ``expert_product``."""
    return _grouped(gradient, weights, ends, out, 1, "gradient")


def expert_weight_gradient(
    gradient: Tensor,
    x: Union[Tensor, ActivationCheckpoint],
    ends: Optional[Tensor],
    *,
    out: Optional[Tensor] = None,
    out_dtype: torch.dtype = torch.float32,
) -> Tensor:
    """``dW_e = sum over e's rows t of dy[t] x[t]^T``: (experts, outputs, inputs), or (outputs, inputs)
    without ``ends``; zeros for an expert without rows.

    ``gradient`` is (tokens, outputs); ``x`` (tokens, inputs) of the same type, or the checkpoint that
    was made from it, which is restored for the time of the call (in memory of its own).  The result is
    float32, the type ``soap_step`` takes, or ``out_dtype`` (the gradient's own type); ``out`` receives it
    instead of a new tensor, in its own type."""
    code = _check_values("gradient", gradient)
    saved = isinstance(x, ActivationCheckpoint)
    if saved:
        _check_checkpoint(x)
        values, exponents, dtype = x
    else:
        _check_values("x", x)
        values, exponents, dtype = x, None, x.dtype
    if dtype != gradient.dtype:
        raise ValueError(f"x must use {gradient.dtype} as gradient does, got {dtype}.")
    (tokens, inputs), (rows, outputs) = values.shape, gradient.shape
    if rows != tokens:
        raise ValueError(f"gradient has {rows} rows, expected {tokens}.")
    if ends is None:
        experts, pointer, shape = 1, 0, (outputs, inputs)
    else:
        _check_matrix("ends", ends, 1)
        experts = ends.numel()
        pointer, shape = _check_ends(ends, experts), (experts, outputs, inputs)
    if out is not None:
        out_code = _check_out(out, shape, _out_types(dtype), gradient=gradient, x=values, exponents=exponents, ends=ends)
    elif out_dtype not in _out_types(dtype):
        raise ValueError(f"out_dtype must be {' or '.join(str(d) for d in _out_types(dtype))}, got {out_dtype}.")
    else:
        out_code = _DTYPES[out_dtype]
    index = gradient.get_device()
    if (index < 0 or values.get_device() != index or (saved and exponents.get_device() != index)
            or (pointer and ends.get_device() != index) or (out is not None and out.get_device() != index)):
        _refuse_devices(gradient.device, gradient=gradient, x=values, exponents=exponents, ends=ends, out=out)
    fresh = out is None
    if fresh:
        out = torch.empty(shape, dtype=out_dtype, device=gradient.device)
    if out.numel() == 0:
        return out
    if saved:
        # (restored for this product alone: expanding the codes inside the product kernel, tile by tile, was
        # slower than reading the matrix once more)
        values = torch.empty((tokens, inputs), dtype=dtype, device=gradient.device)
        if values.numel():
            _launch(index, "soapmi_restore_activations", code, x.codes.data_ptr(), _row_stride(x.codes), exponents.data_ptr(),
                    _row_stride(exponents), tokens, inputs, values.data_ptr(), inputs)
    gradient, ldg = _rows(gradient)
    values, ldx = _rows(values)
    nbytes = 0  # (sums of under 1024 rows are never cut into parts)
    if tokens >= 1024 * experts:
        nbytes = native_library().soapmi_expert_weight_gradient_workspace_bytes(experts, tokens, outputs, inputs)
    work = scratch(nbytes, gradient.device) if nbytes else None
    _launch(index, "soapmi_expert_weight_gradient", code, gradient.data_ptr(), ldg, values.data_ptr(), ldx, pointer, experts,
            tokens, outputs, inputs, out_code, out.data_ptr(), _row_stride(out), out.stride(0) if experts > 1 else 0,
            work.data_ptr() if nbytes else 0, nbytes)
    if not fresh:
        _modified(out)
    return out


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, ends, checkpoint, mixed):
        ctx.dtype, ctx.out_dtype = x.dtype, weights.dtype
        if mixed:
            weights = weights.to(x.dtype)
        y = expert_product(x, weights, ends)
        # each operand is kept for the other's gradient
        needed = weights if ctx.needs_input_grad[0] else None
        kept, exponents = (x if ctx.needs_input_grad[1] else None), None
        if kept is not None and checkpoint:
            kept, exponents, _ = checkpoint_activations(x)
        ctx.save_for_backward(needed, ends, kept, exponents)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gradient):
        weights, ends, kept, exponents = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = expert_input_gradient(gradient, weights, ends)
        if ctx.needs_input_grad[1]:
            x = kept if exponents is None else ActivationCheckpoint(kept, exponents, ctx.dtype)
            dw = expert_weight_gradient(gradient, x, ends, out_dtype=ctx.out_dtype)
        return dx, dw, None, None, None


def expert_linear(x: Tensor, weights: Tensor, ends: Optional[Tensor], *, checkpoint: bool = False) -> Tensor:
    """``expert_product`` for autograd: gradients of ``x`` and ``weights`` come from
    ``expert_input_gradient`` and ``expert_weight_gradient``.

    With ``checkpoint`` the input is kept for the backward pass in 8 bits (``checkpoint_activations``)
    instead of in its own type; the weights' gradient is then that of the restored input, ``x``'s
    gradient and the result are unchanged.

    Under ``torch.autocast`` the product and the gradients are formed in autocast's type.  Weights kept in
    float32 then get their gradient in float32, as the sums are: it is not rounded on the way.

    To capture it with its backward pass into a graph, capture both together and let no earlier autograd
    graph of the same leaves live: torch accumulates a leaf's gradient on the stream of the first graph that
    holds the leaf, and a capture cannot wait for that stream."""
    mixed = False
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        _check_values("x", x)
        _check_values("weights", weights, 2 if ends is None else 3)
        x = x.to(dtype)
        mixed = weights.dtype == torch.float32 != dtype
        if not mixed and weights.dtype != dtype:
            weights = weights.to(dtype)
    return _ExpertLinear.apply(x, weights, ends, checkpoint, mixed)


# ---- activation checkpoints ----------------------------------------------------------------


def _check_checkpoint(checkpoint: ActivationCheckpoint) -> None:
    if not isinstance(checkpoint, ActivationCheckpoint):
        raise ValueError(f"checkpoint must be an ActivationCheckpoint, got {type(checkpoint).__name__}.")
    _check_matrix("codes", checkpoint.codes)
    _check_matrix("exponents", checkpoint.exponents)
    if checkpoint.codes.dtype != torch.int8 or checkpoint.exponents.dtype != torch.uint8:
        raise ValueError(f"codes and exponents must use int8 and uint8, got {checkpoint.codes.dtype} and "
                         f"{checkpoint.exponents.dtype}.")
    if checkpoint.dtype not in _DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {checkpoint.dtype}.")
    rows, columns = checkpoint.codes.shape
    blocks = -(-columns // CHECKPOINT_BLOCK)
    if tuple(checkpoint.exponents.shape) != (rows, blocks):
        raise ValueError(f"exponents has shape {tuple(checkpoint.exponents.shape)}, expected {(rows, blocks)}.")
    for name, tensor in (("codes", checkpoint.codes), ("exponents", checkpoint.exponents)):
        size = tensor.size(1)
        if tensor.numel() and ((size > 1 and tensor.stride(1) != 1) or (rows > 1 and tensor.stride(0) < size)):
            raise ValueError(f"{name} must have contiguous rows.")


def _code_matrix(rows: int, columns: int, device) -> Tensor:
    """int8 rows that start at multiples of 16 bytes."""
    if columns % 16 == 0:
        return torch.empty((rows, columns), dtype=torch.int8, device=device)
    return torch.empty((rows, -(-columns // 16) * 16), dtype=torch.int8, device=device)[:, :columns]


def checkpoint_activations(x: Tensor) -> ActivationCheckpoint:
    """Keep a matrix in 8 bits, with a power-of-two step for each row and 128 columns: half the memory
    of 16-bit activations.  A value is restored to within half a step (within a step above 127.5
    steps), a step being at most 1/64 of the largest magnitude of its 128 columns, or 2^-126 (float16:
    2^-24, its smallest value) where that is more.  128 columns that hold an infinity or NaN are restored
    as NaN."""
    code = _check_values("x", x)
    index = x.get_device()
    if index < 0:
        _refuse_devices(x.device, x=x)
    rows, columns = x.shape
    codes = _code_matrix(rows, columns, x.device)
    exponents = torch.empty((rows, -(-columns // CHECKPOINT_BLOCK)), dtype=torch.uint8, device=x.device)
    if rows and columns:
        values, ldx = _rows(x)
        _launch(index, "soapmi_checkpoint_activations", code, values.data_ptr(), ldx, rows, columns, codes.data_ptr(),
                _row_stride(codes), exponents.data_ptr(), -(-columns // CHECKPOINT_BLOCK))
    return ActivationCheckpoint(codes, exponents, x.dtype)


def restore_activations(checkpoint: ActivationCheckpoint, *, out: Optional[Tensor] = None) -> Tensor:
    """The matrix that a checkpoint stands for, in the type it was made from."""
    _check_checkpoint(checkpoint)
    codes, exponents, dtype = checkpoint
    rows, columns = codes.shape
    if out is not None:
        _check_out(out, (rows, columns), (dtype,), codes=codes, exponents=exponents)
    index = codes.get_device()
    if index < 0 or exponents.get_device() != index or (out is not None and out.get_device() != index):
        _refuse_devices(codes.device, codes=codes, exponents=exponents, out=out)
    fresh = out is None
    if fresh:
        out = torch.empty((rows, columns), dtype=dtype, device=codes.device)
    if rows and columns:
        _launch(index, "soapmi_restore_activations", _DTYPES[dtype], codes.data_ptr(), _row_stride(codes),
                exponents.data_ptr(), _row_stride(exponents), rows, columns, out.data_ptr(), _row_stride(out))
        if not fresh:
            _modified(out)
    return out


# ---- 8-bit integer product -----------------------------------------------------------------


def quantize_tokens(x: Tensor) -> Tuple[Tensor, Tensor]:
    """Codes (int8) and scales (float32, one for each row) of a matrix: scale = largest magnitude / 127,
    code = 127 x / largest magnitude, to the nearest, halves to even.  The rows are tokens, or a weight's
    output channels.
    A row of zeros has scale 0; one that holds an infinity or NaN has scale NaN."""
    code = _check_values("x", x)
    index = x.get_device()
    if index < 0:
        _refuse_devices(x.device, x=x)
    rows, columns = x.shape
    codes = _code_matrix(rows, columns, x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows:
        values, ldx = _rows(x)
        _launch(index, "soapmi_quantize_rows", code, values.data_ptr(), ldx, rows, columns, codes.data_ptr(),
                _row_stride(codes), scales.data_ptr())
    return codes, scales


def _check_codes(name: str, codes: Tensor, scales: Tensor) -> None:
    _check_matrix(name, codes)
    if codes.dtype != torch.int8:
        raise ValueError(f"{name} must use int8, got {codes.dtype}.")
    _check_matrix(f"{name}' scales", scales, 1)
    if scales.dtype != torch.float32:
        raise ValueError(f"{name}' scales must use float32, got {scales.dtype}.")
    rows, count = codes.size(0), scales.numel()
    if count != rows:
        raise ValueError(f"{name} have {rows} rows and {count} scales.")
    if count > 1 and scales.stride(0) != 1:
        raise ValueError(f"{name}' scales must be contiguous.")


def int8_product(
    codes: Tensor,
    scales: Tensor,
    weight_codes: Tensor,
    weight_scales: Tensor,
    *,
    out: Optional[Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
) -> Tensor:
    """``y[t, j] = scales[t] weight_scales[j] sum over i of codes[t, i] weight_codes[j, i]``.

    ``codes`` is (tokens, inputs), ``weight_codes`` (outputs, inputs), both as ``quantize_tokens`` makes
    them from the rows of an activation and of a weight matrix; the integer sum is exact.  The result is
    (tokens, outputs) of ``out_dtype`` (bfloat16, float16 or float32), or goes to ``out``."""
    _check_codes("codes", codes, scales)
    _check_codes("weight_codes", weight_codes, weight_scales)
    tokens, inner = codes.shape
    outputs, width = weight_codes.shape
    if width != inner:
        raise ValueError(f"weight_codes have {width} columns, expected {inner}.")
    if inner > _INT8_MAX_INNER:
        raise ValueError(f"codes have {inner} columns, at most {_INT8_MAX_INNER} keep the integer sums inside 32 bits.")
    if out is not None:
        out_code = _check_out(out, (tokens, outputs), tuple(_DTYPES), codes=codes, scales=scales, weight_codes=weight_codes,
                              weight_scales=weight_scales)
    else:
        out_code = _DTYPES.get(out_dtype)
        if out_code is None:
            raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}.")
    index = codes.get_device()
    if (index < 0 or scales.get_device() != index or weight_codes.get_device() != index
            or weight_scales.get_device() != index or (out is not None and out.get_device() != index)):
        _refuse_devices(codes.device, codes=codes, scales=scales, weight_codes=weight_codes, weight_scales=weight_scales,
                        out=out)
    fresh = out is None
    if fresh:
        out = torch.empty((tokens, outputs), dtype=out_dtype, device=codes.device)
    if tokens and outputs:
        rows, ldq = _rows(codes)
        matrix, ldw = _rows(weight_codes)
        _launch(index, "soapmi_int8_product", rows.data_ptr(), ldq, scales.data_ptr(), matrix.data_ptr(), ldw,
                weight_scales.data_ptr(), tokens, outputs, inner, out_code, out.data_ptr(), _row_stride(out))
        if not fresh:
            _modified(out)
    return out
